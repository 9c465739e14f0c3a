// Group normalisation with an activation over channels-last images, forward and backward.
//
//   mean_g, var_g over the pixels and the C / G channels of group g of one image
//   xhat = (x - mean_g) / sqrt(var_g + eps),   u = w_c xhat + b_c,   y = act(u)
//   du = dy act'(u),   db_c = sum du,   dw_c = sum du xhat
//   dx = rstd_g (w_c du - mean_g(w du) - xhat mean_g(w du xhat))
//
// Both directions are bound by memory: the statistics of a group need all of an image before its first output, so
// x (and dy) is read twice and the result written once.  Images are handled in turns small enough for the second
// read to come from L2 (see images_per_turn).  Three launches per turn: partial sums per chunk of an image, their
// join, and the pass that writes.  Sums are joined in a fixed order, so results do not change from run to run.
//
// Layout of the work: a thread owns V neighbouring values (16 bytes where alignment allows) of a "row" and walks
// down the rows, so that its V channels never change.  A row is one pixel when V divides C; where it does not and
// the pixels are dense, a row is lcm(C, V) values (several pixels), which keeps 16-byte loads for odd C.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace d3gs {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4, kUnroll2 = 2;   // rows in flight per thread: kernels that read x, that read x and dy
constexpr int kCtas = 4, kCtas2 = 3;       // and their CTAs per SM, which the registers are bounded for
constexpr int kMaxChannels = 16384;       // per-channel sums of one CTA stay in shared memory
constexpr int64_t kTurnBytes = 48 << 20;  // inputs of one turn, to be found in L2 (126 MB) by the second pass
constexpr int kJoinThreads = 256, kMaxChunks = 1024;

enum { kActNone = 0, kActSilu = 1, kActGelu = 2 };

template <typename T> __device__ __forceinline__ float to_f(T v) { return (float)v; }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v) { return (T)v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }

// one weight / bias value of any of the three types
__device__ __forceinline__ float load_param(const void* p, int dtype, int i) {
    if (dtype == D3GS_DTYPE_F32) return static_cast<const float*>(p)[i];
    if (dtype == D3GS_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_param(void* p, int dtype, int i, float v) {
    if (dtype == D3GS_DTYPE_F32) static_cast<float*>(p)[i] = v;
    else if (dtype == D3GS_DTYPE_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

template <typename T, int V> struct alignas(sizeof(T) * V) Vec { T v[V]; };

// The logistic function by ex2 and reciprocal of the special-function unit, about 2e-7 relative; u -> -inf gives 0.
__device__ __forceinline__ float logistic(float u) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + __expf(-u)));
    return r;
}

template <int ACT> __device__ __forceinline__ float act_value(float u) {
    if (ACT == kActSilu) return u * logistic(u);
    if (ACT == kActGelu) return 0.5f * u * (1.0f + erff(u * 0.70710678f));
    return u;
}
template <int ACT> __device__ __forceinline__ float act_slope(float u) {
    if (ACT == kActSilu) {
        const float s = logistic(u);
        return s * fmaf(u, 1.0f - s, 1.0f);
    }
    if (ACT == kActGelu) return fmaf(u * 0.39894228f, __expf(-0.5f * u * u), 0.5f * (1.0f + erff(u * 0.70710678f)));
    return 1.0f;
}

// Launches follow one another closely: a kernel may start while its predecessor's last CTAs run, and waits here before
// it touches memory.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

struct Args {
    const void *x, *dy, *weight, *bias;
    void *y, *dweight, *dbias;   // y: output of the forward, dx in the backward
    float* stats;                // [B,G,2] mean, rstd
    float* part;                 // forward [B,G,chunks,2] mean, M2; backward [B,chunks,C,2] sum du, sum du xhat
    float* sums;                 // backward [B,C,2]
    int64_t elems;               // values of one image
    int64_t rows;                // rows of one image (the last may be short)
    int64_t chunk_rows;
    int64_t x_batch, x_row, dy_batch, dy_row, y_batch;   // strides in values
    int batch, chunks, C, G, cpg;
    int L, P;                    // values and vectors per row
    int first;                   // first image of this turn
    int wdtype, act;
    float eps;
};

// What a thread of the walk owns: vector `vec` of rows r0 + lane_row, step rows apart.
struct Walk {
    int rp, lane_row;            // rows the CTA takes at once, this thread's row among them
    bool on;
};
__device__ __forceinline__ Walk make_walk(const Args& a, int tile) {
    Walk w;
    if (a.P <= kThreads) {
        w.rp = kThreads / a.P;
        w.lane_row = threadIdx.x / a.P;
        w.on = w.lane_row < w.rp;
    } else {
        w.rp = 1;
        w.lane_row = 0;
        w.on = tile * kThreads + (int)threadIdx.x < a.P;
    }
    return w;
}
__device__ __forceinline__ int walk_vec(const Args& a, int tile) {
    return a.P <= kThreads ? (int)threadIdx.x % a.P : tile * kThreads + (int)threadIdx.x;
}

// Rows of [r0, r1) in which vector `vec` is whole, and how many of its values the row after them holds (0: none).
template <int V> __device__ __forceinline__ int64_t whole_rows(const Args& a, int64_t r1, int vec, int& tail) {
    tail = 0;
    if (r1 < a.rows) return r1;
    const int64_t left = a.elems - (a.rows - 1) * (int64_t)a.L - (int64_t)vec * V;   // in the last row, from this vector on
    if (left >= V) return r1;
    tail = left > 0 ? (int)left : 0;
    return r1 - 1;
}

// ---- forward, pass 1: mean and centred square sum of every group over one chunk of one image ----------------------
// Squares are taken around the mean k of the thread's first rows: when k is far from the mean of the rest, the rows
// that k came from are themselves far from it and the variance is at least kUnroll/n of that distance squared, so
// the cancellation in q - s^2/n costs at most n/kUnroll units of the last place, whatever the mean.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads, kCtas) gn_stats_kernel(const Args a) {
    extern __shared__ float sh[];
    let_next_start();
    wait_for_previous();
    const int b = a.first + blockIdx.y, chunk = blockIdx.x;
    const int64_t r0 = chunk * a.chunk_rows, r1 = min(a.rows, r0 + a.chunk_rows);
    const T* x = static_cast<const T*>(a.x) + b * a.x_batch;
    const int slots = (a.P <= kThreads ? kThreads / a.P : 1) * a.L;   // entries of the CTA: [row][value of the row]
    float *s_n = sh, *s_mean = sh + slots, *s_m2 = sh + 2 * slots;
    const int tiles = a.P <= kThreads ? 1 : (a.P + kThreads - 1) / kThreads;
    for (int tile = 0; tile < tiles; ++tile) {
        const Walk w = make_walk(a, tile);
        if (!w.on) continue;
        const int vec = walk_vec(a, tile);
        int tail;
        const int64_t end = whole_rows<V>(a, r1, vec, tail);
        const T* p = x + (int64_t)vec * V;
        float k[V], s[V], q[V];
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = q[j] = k[j] = 0.0f;
        int64_t r = r0 + w.lane_row;
        const int64_t step = w.rp * a.x_row;
        p += r * a.x_row;
        const int got = r < end ? (int)min((int64_t)kUnroll, (end - r + w.rp - 1) / w.rp) : 0;
        for (int u = 0; u < got; ++u) {
            const Vec<T, V> f = *reinterpret_cast<const Vec<T, V>*>(p + u * step);
#pragma unroll
            for (int j = 0; j < V; ++j) k[j] += to_f(f.v[j]);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) k[j] /= (float)max(got, 1);
        auto add = [&](const Vec<T, V>& x) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = to_f(x.v[j]) - k[j];
                s[j] += d;
                q[j] = fmaf(d, d, q[j]);
            }
        };
        int n = 0;
        for (; r + (kUnroll - 1) * w.rp < end; r += kUnroll * w.rp, p += kUnroll * step, n += kUnroll) {
            Vec<T, V> v[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) v[u] = *reinterpret_cast<const Vec<T, V>*>(p + u * step);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) add(v[u]);
        }
        for (; r < end; r += w.rp, p += step, ++n) add(*reinterpret_cast<const Vec<T, V>*>(p));
        // the short row at the image's end belongs to the thread whose turn it is
        const bool mine = tail > 0 && end >= r0 && (end - r0) % w.rp == w.lane_row;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            int nj = n;
            if (mine && j < tail) {
                const float v = to_f(p[j]);   // r == end
                if (n == 0) k[j] = v;
                const float d = v - k[j];
                s[j] += d;
                q[j] = fmaf(d, d, q[j]);
                nj = n + 1;
            }
            const float mean = nj > 0 ? s[j] / nj : 0.0f;
            const float m2 = q[j] - s[j] * mean;
            const int e = w.lane_row * a.L + vec * V + j;
            s_n[e] = (float)nj;
            s_mean[e] = k[j] + mean;
            s_m2[e] = m2 < 0.0f ? 0.0f : m2;      // not fmaxf: a NaN stays one
        }
    }
    __syncthreads();
    // one warp per group joins its entries: first the mean, then the squares around it
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int pixels = slots / a.C, items = pixels * a.cpg;
    for (int g = warp; g < a.G; g += kThreads / 32) {
        const float near = s_mean[g * a.cpg];   // a value of the group's size: differences from it are added up
        float n = 0.0f, t = 0.0f;
        for (int i = lane; i < items; i += 32) {
            const int e = (i / a.cpg) * a.C + g * a.cpg + i % a.cpg;
            n += s_n[e];
            if (s_n[e] > 0.0f) t = fmaf(s_n[e], s_mean[e] - near, t);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            n += __shfl_xor_sync(~0u, n, o);
            t += __shfl_xor_sync(~0u, t, o);
        }
        const float mean = n > 0.0f ? near + t / n : 0.0f;
        float m2 = 0.0f;
        for (int i = lane; i < items; i += 32) {
            const int e = (i / a.cpg) * a.C + g * a.cpg + i % a.cpg;
            if (s_n[e] > 0.0f) {
                const float d = s_mean[e] - mean;
                m2 += fmaf(s_n[e] * d, d, s_m2[e]);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m2 += __shfl_xor_sync(~0u, m2, o);
        if (lane == 0) {
            float* out = a.part + (((int64_t)b * a.G + g) * a.chunks + chunk) * 2;
            out[0] = mean;
            out[1] = m2;
        }
    }
}

// values of one group in one chunk
__device__ __forceinline__ float chunk_count(const Args& a, int chunk) {
    const int64_t e0 = chunk * a.chunk_rows * a.L, e1 = min(a.elems, (chunk + 1) * a.chunk_rows * a.L);
    return (float)((e1 - e0) / a.C * a.cpg);
}

// ---- forward, join: one CTA per (image, group) over the chunks ----------------------------------------------------
__device__ __forceinline__ float cta_sum(float v, float* sh) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int k = 0; k < kJoinThreads / 32; ++k) v += sh[k];
    return v;
}
__global__ void __launch_bounds__(kJoinThreads) gn_stats_join_kernel(const Args a) {
    __shared__ float sh[2][kJoinThreads / 32];
    let_next_start();
    wait_for_previous();
    const int64_t bg = (int64_t)a.first * a.G + blockIdx.x;
    const float2* part = reinterpret_cast<const float2*>(a.part) + bg * a.chunks;
    const float total = (float)(a.elems / a.C * a.cpg), near = part[0].x;
    float2 mine[kMaxChunks / kJoinThreads];
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < kMaxChunks / kJoinThreads; ++i) {
        const int k = threadIdx.x + i * kJoinThreads;
        mine[i] = k < a.chunks ? part[k] : make_float2(near, 0.0f);
    }
#pragma unroll
    for (int i = 0; i < kMaxChunks / kJoinThreads; ++i) {
        const int k = threadIdx.x + i * kJoinThreads;
        if (k < a.chunks) t = fmaf(chunk_count(a, k) / total, mine[i].x - near, t);
    }
    const float mean = near + cta_sum(t, sh[0]);
    float m2 = 0.0f;
#pragma unroll
    for (int i = 0; i < kMaxChunks / kJoinThreads; ++i) {
        const int k = threadIdx.x + i * kJoinThreads;
        if (k < a.chunks) {
            const float d = mine[i].x - mean;
            m2 += fmaf(chunk_count(a, k) * d, d, mine[i].y);
        }
    }
    m2 = cta_sum(m2, sh[1]);
    if (threadIdx.x == 0) {
        a.stats[bg * 2] = mean;
        a.stats[bg * 2 + 1] = 1.0f / sqrtf(m2 / total + a.eps);
    }
}

// mean, rstd, weight and bias of channel `ch` of image b
__device__ __forceinline__ float4 load_coef(const Args& a, int b, int ch) {
    const float2 st = reinterpret_cast<const float2*>(a.stats)[(int64_t)b * a.G + ch / a.cpg];
    return make_float4(st.x, st.y, a.weight ? load_param(a.weight, a.wdtype, ch) : 1.0f,
                       a.bias ? load_param(a.bias, a.wdtype, ch) : 0.0f);
}

// ---- forward, pass 2 -----------------------------------------------------------------------------------------------
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads, kCtas) gn_apply_kernel(const Args a) {
    let_next_start();
    wait_for_previous();
    const int b = a.first + blockIdx.y, chunk = a.chunks - 1 - blockIdx.x;   // last read first: still in L2
    const int64_t r0 = chunk * a.chunk_rows, r1 = min(a.rows, r0 + a.chunk_rows);
    const T* x = static_cast<const T*>(a.x) + b * a.x_batch;
    T* y = static_cast<T*>(a.y) + b * a.y_batch;
    const int tiles = a.P <= kThreads ? 1 : (a.P + kThreads - 1) / kThreads;
    for (int tile = 0; tile < tiles; ++tile) {
        const Walk w = make_walk(a, tile);
        if (!w.on) continue;
        const int vec = walk_vec(a, tile);
        int tail;
        const int64_t end = whole_rows<V>(a, r1, vec, tail);
        float k[V], q[V];   // u = k x + q; q is rounded at the size of mean rstd, as mean itself is
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float4 c = load_coef(a, b, (vec * V + j) % a.C);
            k[j] = c.y * c.z;
            q[j] = fmaf(-c.x, k[j], c.w);
        }
        auto value = [&](T v, int j) { return from_f<T>(act_value<ACT>(fmaf(to_f(v), k[j], q[j]))); };
        int64_t r = r0 + w.lane_row;
        const T* p = x + r * a.x_row + (int64_t)vec * V;
        T* o = y + r * a.L + (int64_t)vec * V;
        const int64_t step = w.rp * a.x_row, ostep = (int64_t)w.rp * a.L;
        auto write = [&](T* to, const Vec<T, V>& v) {
            Vec<T, V> res;
#pragma unroll
            for (int j = 0; j < V; ++j) res.v[j] = value(v.v[j], j);
            *reinterpret_cast<Vec<T, V>*>(to) = res;
        };
        for (; r + (kUnroll - 1) * w.rp < end; r += kUnroll * w.rp, p += kUnroll * step, o += kUnroll * ostep) {
            Vec<T, V> v[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) v[u] = *reinterpret_cast<const Vec<T, V>*>(p + u * step);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) write(o + u * ostep, v[u]);
        }
        for (; r < end; r += w.rp, p += step, o += ostep) write(o, *reinterpret_cast<const Vec<T, V>*>(p));
        if (tail > 0 && end >= r0 && (end - r0) % w.rp == w.lane_row)   // r == end: the short row
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j < tail) o[j] = value(p[j], j);
    }
}

// ---- backward, pass 1: sum of du and of du xhat per channel over one chunk ----------------------------------------
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads, kCtas2) gn_grad_sums_kernel(const Args a) {
    extern __shared__ float sh[];
    let_next_start();
    wait_for_previous();
    const int b = a.first + blockIdx.y, chunk = blockIdx.x;
    const int64_t r0 = chunk * a.chunk_rows, r1 = min(a.rows, r0 + a.chunk_rows);
    const T* x = static_cast<const T*>(a.x) + b * a.x_batch;
    const T* dy = static_cast<const T*>(a.dy) + b * a.dy_batch;
    const int slots = (a.P <= kThreads ? kThreads / a.P : 1) * a.L;
    float *s_1 = sh, *s_2 = sh + slots;
    const int tiles = a.P <= kThreads ? 1 : (a.P + kThreads - 1) / kThreads;
    for (int tile = 0; tile < tiles; ++tile) {
        const Walk w = make_walk(a, tile);
        if (!w.on) continue;
        const int vec = walk_vec(a, tile);
        int tail;
        const int64_t end = whole_rows<V>(a, r1, vec, tail);
        float mean[V], k[V], q[V], s1[V], s2[V];   // u = k (x - mean) + q; s2 sums du (x - mean)
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float4 c = load_coef(a, b, (vec * V + j) % a.C);
            mean[j] = c.x;
            k[j] = c.y * c.z;
            q[j] = c.w;
            s1[j] = s2[j] = 0.0f;
        }
        auto add = [&](T xv, T dv, int j) {
            const float d = to_f(xv) - mean[j];
            const float du = to_f(dv) * act_slope<ACT>(fmaf(d, k[j], q[j]));
            s1[j] += du;
            s2[j] = fmaf(du, d, s2[j]);
        };
        int64_t r = r0 + w.lane_row;
        const T* p = x + r * a.x_row + (int64_t)vec * V;
        const T* d = dy + r * a.dy_row + (int64_t)vec * V;
        const int64_t step = w.rp * a.x_row, dstep = w.rp * a.dy_row;
        for (; r + (kUnroll2 - 1) * w.rp < end; r += kUnroll2 * w.rp, p += kUnroll2 * step, d += kUnroll2 * dstep) {
            Vec<T, V> v[kUnroll2], g[kUnroll2];
#pragma unroll
            for (int u = 0; u < kUnroll2; ++u) {
                v[u] = *reinterpret_cast<const Vec<T, V>*>(p + u * step);
                g[u] = *reinterpret_cast<const Vec<T, V>*>(d + u * dstep);
            }
#pragma unroll
            for (int u = 0; u < kUnroll2; ++u)
#pragma unroll
                for (int j = 0; j < V; ++j) add(v[u].v[j], g[u].v[j], j);
        }
        for (; r < end; r += w.rp, p += step, d += dstep) {
            const Vec<T, V> v = *reinterpret_cast<const Vec<T, V>*>(p), g = *reinterpret_cast<const Vec<T, V>*>(d);
#pragma unroll
            for (int j = 0; j < V; ++j) add(v.v[j], g.v[j], j);
        }
        const bool mine = tail > 0 && end >= r0 && (end - r0) % w.rp == w.lane_row;   // r == end: the short row
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (mine && j < tail) add(p[j], d[j], j);
            s_1[w.lane_row * a.L + vec * V + j] = s1[j];
            s_2[w.lane_row * a.L + vec * V + j] = s2[j] * load_coef(a, b, (vec * V + j) % a.C).y;
        }
    }
    __syncthreads();
    float2* out = reinterpret_cast<float2*>(a.part) + ((int64_t)b * a.chunks + chunk) * a.C;
    for (int ch = threadIdx.x; ch < a.C; ch += kThreads) {
        float t1 = 0.0f, t2 = 0.0f;
        for (int e = ch; e < slots; e += a.C) {
            t1 += s_1[e];
            t2 += s_2[e];
        }
        out[ch] = make_float2(t1, t2);
    }
}

// ---- backward, join: sums of every (image, channel) over the chunks; 16 channels x 64 lanes per CTA ---------------
__global__ void __launch_bounds__(1024) gn_grad_join_kernel(const Args a) {
    __shared__ float2 sh[64][16];
    let_next_start();
    wait_for_previous();
    const int in = threadIdx.x & 15, ch = blockIdx.x * 16 + in, part = threadIdx.x >> 4, b = a.first + blockIdx.y;
    float2 t = make_float2(0.0f, 0.0f);
    if (ch < a.C) {
        const float2* p = reinterpret_cast<const float2*>(a.part) + (int64_t)b * a.chunks * a.C + ch;
#pragma unroll 4
        for (int k = part; k < a.chunks; k += 64) {
            const float2 v = p[(int64_t)k * a.C];
            t.x += v.x;
            t.y += v.y;
        }
    }
    sh[part][in] = t;
    __syncthreads();
#pragma unroll
    for (int half = 32; half > 0; half >>= 1) {
        if (part < half) {
            sh[part][in].x += sh[part + half][in].x;
            sh[part][in].y += sh[part + half][in].y;
        }
        __syncthreads();
    }
    if (part == 0 && ch < a.C) reinterpret_cast<float2*>(a.sums)[(int64_t)b * a.C + ch] = sh[0][in];
}

// ---- backward, pass 2: dx, and (last turn) the parameter gradients ------------------------------------------------
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads, kCtas2) gn_grad_apply_kernel(const Args a, int params) {
    extern __shared__ float sh[];   // [G][2] group means of w du and w du xhat
    let_next_start();
    wait_for_previous();
    const int b = a.first + blockIdx.y, chunk = a.chunks - 1 - blockIdx.x;
    const float2* sums = reinterpret_cast<const float2*>(a.sums);
    const float inv = 1.0f / (float)(a.elems / a.C * a.cpg);
    for (int g = threadIdx.x >> 5; g < a.G; g += kThreads / 32) {
        float m1 = 0.0f, m2 = 0.0f;
        for (int i = threadIdx.x & 31; i < a.cpg; i += 32) {
            const int ch = g * a.cpg + i;
            const float2 s = sums[(int64_t)b * a.C + ch];
            const float w = a.weight ? load_param(a.weight, a.wdtype, ch) : 1.0f;
            m1 = fmaf(w, s.x, m1);
            m2 = fmaf(w, s.y, m2);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            m1 += __shfl_xor_sync(~0u, m1, o);
            m2 += __shfl_xor_sync(~0u, m2, o);
        }
        if ((threadIdx.x & 31) == 0) {
            sh[g * 2] = m1 * inv;
            sh[g * 2 + 1] = m2 * inv;
        }
    }
    if (params && blockIdx.y == 0)   // every CTA of one image takes a share of the channels
        for (int ch = blockIdx.x * kThreads + threadIdx.x; ch < a.C; ch += gridDim.x * kThreads) {
            float t1 = 0.0f, t2 = 0.0f;
            for (int k = 0; k < a.batch; ++k) {
                const float2 s = sums[(int64_t)k * a.C + ch];
                t1 += s.x;
                t2 += s.y;
            }
            if (a.dweight) store_param(a.dweight, a.wdtype, ch, t2);
            if (a.dbias) store_param(a.dbias, a.wdtype, ch, t1);
        }
    __syncthreads();
    if (!a.y) return;
    const int64_t r0 = chunk * a.chunk_rows, r1 = min(a.rows, r0 + a.chunk_rows);
    const T* x = static_cast<const T*>(a.x) + b * a.x_batch;
    const T* dy = static_cast<const T*>(a.dy) + b * a.dy_batch;
    T* dx = static_cast<T*>(a.y) + b * a.y_batch;
    const int tiles = a.P <= kThreads ? 1 : (a.P + kThreads - 1) / kThreads;
    for (int tile = 0; tile < tiles; ++tile) {
        const Walk w = make_walk(a, tile);
        if (!w.on) continue;
        const int vec = walk_vec(a, tile);
        int tail;
        const int64_t end = whole_rows<V>(a, r1, vec, tail);
        float k[V], q[V], kx[V], kc[V];   // u = k x + q, dx = k du + kx x + kc
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int ch = (vec * V + j) % a.C;
            const float4 c = load_coef(a, b, ch);
            const float m1 = sh[ch / a.cpg * 2], m2 = sh[ch / a.cpg * 2 + 1];
            k[j] = c.y * c.z;
            q[j] = fmaf(-c.x, k[j], c.w);
            kx[j] = -c.y * c.y * m2;
            kc[j] = fmaf(-c.x, kx[j], -c.y * m1);
        }
        auto value = [&](T xv, T dv, int j) {
            const float x = to_f(xv), du = to_f(dv) * act_slope<ACT>(fmaf(x, k[j], q[j]));
            return from_f<T>(fmaf(k[j], du, fmaf(kx[j], x, kc[j])));
        };
        int64_t r = r0 + w.lane_row;
        const T* p = x + r * a.x_row + (int64_t)vec * V;
        const T* d = dy + r * a.dy_row + (int64_t)vec * V;
        T* o = dx + r * a.L + (int64_t)vec * V;
        const int64_t step = w.rp * a.x_row, dstep = w.rp * a.dy_row, ostep = (int64_t)w.rp * a.L;
        auto write = [&](T* to, const Vec<T, V>& v, const Vec<T, V>& g) {
            Vec<T, V> res;
#pragma unroll
            for (int j = 0; j < V; ++j) res.v[j] = value(v.v[j], g.v[j], j);
            *reinterpret_cast<Vec<T, V>*>(to) = res;
        };
        for (; r + (kUnroll2 - 1) * w.rp < end; r += kUnroll2 * w.rp, p += kUnroll2 * step, d += kUnroll2 * dstep, o += kUnroll2 * ostep) {
            Vec<T, V> v[kUnroll2], g[kUnroll2];
#pragma unroll
            for (int u = 0; u < kUnroll2; ++u) {
                v[u] = *reinterpret_cast<const Vec<T, V>*>(p + u * step);
                g[u] = *reinterpret_cast<const Vec<T, V>*>(d + u * dstep);
            }
#pragma unroll
            for (int u = 0; u < kUnroll2; ++u) write(o + u * ostep, v[u], g[u]);
        }
        for (; r < end; r += w.rp, p += step, d += dstep, o += ostep)
            write(o, *reinterpret_cast<const Vec<T, V>*>(p), *reinterpret_cast<const Vec<T, V>*>(d));
        if (tail > 0 && end >= r0 && (end - r0) % w.rp == w.lane_row)   // r == end: the short row
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j < tail) o[j] = value(p[j], d[j], j);
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------
int gcd(int64_t a, int64_t b) {
    while (b) {
        const int64_t t = a % b;
        a = b;
        b = t;
    }
    return (int)a;
}
int elem_size(int dtype) { return dtype == D3GS_DTYPE_F32 ? 4 : 2; }

// The widest vector with which every row of every tensor starts on a multiple of its size.
int pick_vector(const D3gsGroupNorm& d, const void* x, const void* dy, const void* out, bool backward) {
    const int size = elem_size(d.dtype);
    for (int v = 16 / size; v > 1; v /= 2) {
        const bool flat = d.x_pixel_stride == d.channels && (!backward || d.dy_pixel_stride == d.channels);
        const int p = d.channels / gcd(d.channels, v);
        if (d.channels % v != 0 && (!flat || p > kThreads)) continue;
        uint64_t bad = (uintptr_t)x | (uintptr_t)out | (uintptr_t)dy;
        if (d.batch > 1)
            bad |= (uint64_t)(d.pixels * d.channels * size) | (uint64_t)(d.x_batch_stride * size) |
                   (backward ? (uint64_t)(d.dy_batch_stride * size) : 0);
        if (d.channels % v == 0)
            bad |= (uint64_t)(d.x_pixel_stride * size) | (backward ? (uint64_t)(d.dy_pixel_stride * size) : 0);
        if (bad % (uint64_t)(v * size) == 0) return v;
    }
    return 1;
}

// Images per turn: as many as keep the turn's inputs within kTurnBytes, at least one.
int images_per_turn(const D3gsGroupNorm& d, bool backward) {
    const int64_t image = d.pixels * d.channels * elem_size(d.dtype) * (backward ? 2 : 1);
    int64_t n = kTurnBytes / (image > 0 ? image : 1);
    if (n > d.batch) n = d.batch;
    return (int)(n < 1 ? 1 : n);
}

// Chunks of one image: as many CTAs in a turn as run at once, none with less than two vectors a thread.
int chunks_of(const D3gsGroupNorm& d, bool backward) {
    const int turn = images_per_turn(d, backward);
    const int64_t want = div_up64((backward ? kCtas2 : kCtas) * 148, turn), values = d.pixels * d.channels;
    const int64_t most = div_up64(values, (int64_t)kThreads * (16 / elem_size(d.dtype)) * 2);
    int64_t n = want < most ? want : most;
    return (int)(n < 1 ? 1 : n > kMaxChunks ? kMaxChunks : n);
}

int32_t check(const D3gsGroupNorm* d, const char* what) {
    D3GS_REQUIRE(d != nullptr, "%s: desc is NULL", what);
    D3GS_REQUIRE(d->batch >= 0 && d->batch <= 65535 && d->pixels >= 0, "%s: batch %lld (at most 65535), pixels %lld", what,
                 (long long)d->batch, (long long)d->pixels);
    D3GS_REQUIRE(d->channels >= 1 && d->channels <= kMaxChannels, "%s: %d channels (1 to %d)", what, d->channels, kMaxChannels);
    D3GS_REQUIRE(d->groups >= 1 && d->channels % d->groups == 0, "%s: %d groups do not divide %d channels", what, d->groups,
                 d->channels);
    D3GS_REQUIRE(d->pixels <= (int64_t)1 << 40, "%s: image too large", what);
    D3GS_REQUIRE(d->dtype >= 0 && d->dtype <= 2 && d->weight_dtype >= 0 && d->weight_dtype <= 2, "%s: dtype %d / %d", what,
                 d->dtype, d->weight_dtype);
    D3GS_REQUIRE(d->act >= 0 && d->act <= 2, "%s: act %d", what, d->act);
    D3GS_REQUIRE(d->eps >= 0.0f, "%s: eps must not be negative", what);
    return D3GS_OK;
}

struct Workspace {
    size_t part, sums, bytes;   // offsets, total
};
Workspace workspace_of(const D3gsGroupNorm& d, bool backward) {
    Workspace w;
    const size_t chunks = chunks_of(d, backward);
    w.part = 0;
    const size_t n = (size_t)d.batch * chunks * (backward ? d.channels : d.groups) * 8;
    w.sums = (n + 255) / 256 * 256;
    w.bytes = w.sums + (backward ? (size_t)d.batch * d.channels * 8 : 0) + 256;
    return w;
}

Args make_args(const D3gsGroupNorm& d, int v, bool backward, void* ws) {
    Args a{};
    const Workspace w = workspace_of(d, backward);
    a.C = d.channels;
    a.G = d.groups;
    a.cpg = d.channels / d.groups;
    a.elems = d.pixels * d.channels;
    a.P = d.channels / gcd(d.channels, v);             // vectors after which the channels repeat
    a.L = a.P * v;
    a.rows = div_up64(a.elems, a.L);
    a.chunks = chunks_of(d, backward);
    a.chunk_rows = div_up64(a.rows, a.chunks);
    a.chunks = (int)div_up64(a.rows, a.chunk_rows);    // no empty chunk
    a.x_batch = d.x_batch_stride;
    a.dy_batch = d.dy_batch_stride;
    a.x_row = a.L == a.C ? d.x_pixel_stride : a.L;
    a.dy_row = a.L == a.C ? d.dy_pixel_stride : a.L;
    a.y_batch = a.elems;
    a.batch = (int)d.batch;
    a.wdtype = d.weight_dtype;
    a.act = d.act;
    a.eps = d.eps;
    a.part = reinterpret_cast<float*>(static_cast<char*>(ws) + w.part);
    a.sums = reinterpret_cast<float*>(static_cast<char*>(ws) + w.sums);
    return a;
}

template <typename K, typename... A>
int32_t launch(K kernel, const char* name, dim3 grid, unsigned threads, size_t smem, cudaStream_t st, const A&... args) {
    if (smem > 48 * 1024) D3GS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cudaLaunchConfig_t c{};
    c.gridDim = grid;
    c.blockDim = dim3(threads);
    c.dynamicSmemBytes = smem;
    c.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &attr;
    c.numAttrs = 1;
    D3GS_CUDA(cudaLaunchKernelEx(&c, kernel, args...));
    D3GS_LAUNCH_CHECK(name);
    return D3GS_OK;
}

template <typename T, int V, int ACT>
int32_t run_forward(const D3gsGroupNorm& d, Args a, cudaStream_t st) {
    const int turn = images_per_turn(d, false);
    const size_t slots = (size_t)(a.P <= kThreads ? kThreads / a.P : 1) * a.L;
    for (int b = 0; b < a.batch; b += turn) {
        const int images = b + turn <= a.batch ? turn : a.batch - b;
        a.first = b;
        const dim3 grid(a.chunks, images);
        if (int32_t rc = launch(gn_stats_kernel<T, V>, "gn_stats_kernel", grid, kThreads, slots * 12, st, a)) return rc;
        if (int32_t rc = launch(gn_stats_join_kernel, "gn_stats_join_kernel", dim3(images * a.G), kJoinThreads, 0, st, a)) return rc;
        if (int32_t rc = launch(gn_apply_kernel<T, V, ACT>, "gn_apply_kernel", grid, kThreads, 0, st, a)) return rc;
    }
    return D3GS_OK;
}

template <typename T, int V, int ACT>
int32_t run_backward(const D3gsGroupNorm& d, Args a, cudaStream_t st) {
    const int turn = images_per_turn(d, true);
    const size_t slots = (size_t)(a.P <= kThreads ? kThreads / a.P : 1) * a.L;
    for (int b = 0; b < a.batch; b += turn) {
        const int images = b + turn <= a.batch ? turn : a.batch - b;
        a.first = b;
        const dim3 grid(a.chunks, images);
        if (int32_t rc = launch(gn_grad_sums_kernel<T, V, ACT>, "gn_grad_sums_kernel", grid, kThreads, slots * 8, st, a)) return rc;
        if (int32_t rc = launch(gn_grad_join_kernel, "gn_grad_join_kernel", dim3((a.C + 15) / 16, images), 1024, 0, st, a)) return rc;
        const int params = b + images == a.batch && (a.dweight || a.dbias);
        if (int32_t rc = launch(gn_grad_apply_kernel<T, V, ACT>, "gn_grad_apply_kernel", grid, kThreads, (size_t)a.G * 8, st, a, params))
            return rc;
    }
    return D3GS_OK;
}

template <typename T, int V> int32_t run_act(const D3gsGroupNorm& d, const Args& a, bool backward, cudaStream_t st) {
    switch (d.act) {
        case kActNone: return backward ? run_backward<T, V, kActNone>(d, a, st) : run_forward<T, V, kActNone>(d, a, st);
        case kActSilu: return backward ? run_backward<T, V, kActSilu>(d, a, st) : run_forward<T, V, kActSilu>(d, a, st);
        default: return backward ? run_backward<T, V, kActGelu>(d, a, st) : run_forward<T, V, kActGelu>(d, a, st);
    }
}
template <typename T> int32_t run_vec(const D3gsGroupNorm& d, const Args& a, int v, bool backward, cudaStream_t st) {
    switch (v) {
        case 8: if constexpr (sizeof(T) == 2) return run_act<T, 8>(d, a, backward, st);
        case 4: return run_act<T, 4>(d, a, backward, st);
        case 2: return run_act<T, 2>(d, a, backward, st);
        default: return run_act<T, 1>(d, a, backward, st);
    }
}
int32_t run(const D3gsGroupNorm& d, const Args& a, int v, bool backward, void* stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (d.dtype) {
        case D3GS_DTYPE_F32: return run_vec<float>(d, a, v, backward, st);
        case D3GS_DTYPE_BF16: return run_vec<__nv_bfloat16>(d, a, v, backward, st);
        default: return run_vec<__half>(d, a, v, backward, st);
    }
}

}  // namespace
}  // namespace d3gs

using namespace d3gs;

extern "C" size_t d3gs_group_norm_workspace_bytes(const D3gsGroupNorm* desc, int32_t backward) {
    if (check(desc, "d3gs_group_norm_workspace_bytes") != D3GS_OK) return 0;
    return workspace_of(*desc, backward != 0).bytes;
}

extern "C" int32_t d3gs_group_norm_forward(const D3gsGroupNorm* desc, const void* x, const void* weight, const void* bias,
                                           void* y, float* stats, void* ws, size_t ws_bytes, void* stream) {
    if (int32_t rc = check(desc, "d3gs_group_norm_forward")) return rc;
    if (desc->batch == 0 || desc->pixels == 0) return D3GS_OK;
    D3GS_REQUIRE(x && y && stats, "d3gs_group_norm_forward: x, y or stats is NULL");
    D3GS_REQUIRE(ws && ((uintptr_t)ws & 15) == 0 && ws_bytes >= workspace_of(*desc, false).bytes,
                 "d3gs_group_norm_forward: workspace missing, unaligned or smaller than d3gs_group_norm_workspace_bytes");
    const int v = pick_vector(*desc, x, nullptr, y, false);
    Args a = make_args(*desc, v, false, ws);
    a.x = x;
    a.weight = weight;
    a.bias = bias;
    a.y = y;
    a.stats = stats;
    return run(*desc, a, v, false, stream);
}

extern "C" int32_t d3gs_group_norm_backward(const D3gsGroupNorm* desc, const void* x, const void* weight, const void* bias,
                                            const float* stats, const void* dy, void* dx, void* dweight, void* dbias,
                                            void* ws, size_t ws_bytes, void* stream) {
    if (int32_t rc = check(desc, "d3gs_group_norm_backward")) return rc;
    if (desc->batch == 0 || desc->pixels == 0) return D3GS_OK;
    D3GS_REQUIRE(x && dy && stats, "d3gs_group_norm_backward: x, dy or stats is NULL");
    D3GS_REQUIRE(dx || dweight || dbias, "d3gs_group_norm_backward: no gradient is asked for");
    D3GS_REQUIRE(ws && ((uintptr_t)ws & 15) == 0 && ws_bytes >= workspace_of(*desc, true).bytes,
                 "d3gs_group_norm_backward: workspace missing, unaligned or smaller than d3gs_group_norm_workspace_bytes");
    const int v = pick_vector(*desc, x, dy, dx, true);
    Args a = make_args(*desc, v, true, ws);
    a.x = x;
    a.dy = dy;
    a.weight = weight;
    a.bias = bias;
    a.y = dx;
    a.dweight = dweight;
    a.dbias = dbias;
    a.stats = const_cast<float*>(stats);
    return run(*desc, a, v, true, stream);
}

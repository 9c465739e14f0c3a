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
// join, and the pass that writes; one launch for small images, a CTA each (see one_cta).  Sums are joined in a fixed
// order, so results do not change from run to run.
//
// Measured: 1080p x 32 channels in fp16, forward 88 us (133 MB read twice, the second time partly from L2, and written; a
// copy of that size takes 44 us, a plain read 30).  Forward and backward of 4 x 1080p x 32 in bf16 867 us, 4.9 TB/s with
// the second reads, which miss L2 there; of 8 x 135 x 240 x 256 in fp16 263 us, the second reads from L2.
//
// Layout of the work: a thread owns V neighbouring values (16 bytes where alignment allows) of a "row" and walks
// down the rows, so that its V channels never change.  A row is one pixel when V divides C; where it does not and
// the pixels are dense, a row is lcm(C, V) values (several pixels), which keeps 16-byte loads for odd C.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace d3gs {
namespace {

constexpr int kThreads = 256;
// Rows in flight per thread in the kernels that read x, and in those that read x and dy, and their CTAs per SM, which
// the registers are bounded for.  Few CTAs with many loads each do better than many with few: 4 x 1080p x 32 channels
// in 16 bits, forward 413 us with 4 rows and 4 CTAs, 343 us with 8 and 2; backward 664 us with 2 and 3, 544 with 4 and 2.
constexpr int kUnroll = 8, kUnroll2 = 4;
constexpr int kCtas = 2, kCtas2 = 2;
constexpr int kMaxChannels = 16384;       // per-channel sums of one CTA stay in shared memory
constexpr int64_t kTurnBytes = 72 << 20;  // inputs of one turn, to be found in L2 (126 MB) by the second pass
constexpr int kSmall = 4096, kSmallGrad = 2048, kSmallMany = 32768;   // vectors of an image, see one_cta()
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

// ---- values in pairs: the packed 32-bit operations of sm_100 take two per instruction -----------------------------
typedef unsigned long long Two;
__device__ __forceinline__ Two two(float a, float b) {
    Two r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ Two both(float a) { return two(a, a); }
__device__ __forceinline__ float2 split(Two v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
    Two r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
    Two r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// V neighbouring values as they lie in memory; `pair(i)` gives values 2 i and 2 i + 1 (a single value comes twice).
template <typename T, int V> struct alignas(sizeof(T) * V) Vec {
    T v[V];
    __device__ __forceinline__ Two pair(int i) const {
        if constexpr (V == 1) return both(to_f(v[0]));
        else if constexpr (sizeof(T) == 4) return two(to_f(v[2 * i]), to_f(v[2 * i + 1]));
        else {
            const uint32_t w = reinterpret_cast<const uint32_t*>(v)[i];
            if constexpr (std::is_same_v<T, __nv_bfloat16>) return two(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
            else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
                return two(f.x, f.y);
            }
        }
    }
    __device__ __forceinline__ void set(int i, Two x) {
        const float2 f = split(x);
        if constexpr (V == 1) v[0] = from_f<T>(f.x);
        else if constexpr (std::is_same_v<T, __nv_bfloat16>) reinterpret_cast<__nv_bfloat162*>(v)[i] = __floats2bfloat162_rn(f.x, f.y);
        else if constexpr (std::is_same_v<T, __half>) reinterpret_cast<__half2*>(v)[i] = __floats2half2_rn(f.x, f.y);
        else {
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
};
// The first pass over an image reads it plainly, for the second to find in L2; what the second reads and writes is not
// looked at again and should not drive the rest out.
template <typename T, int V> __device__ __forceinline__ Vec<T, V> load(const T* p) { return *reinterpret_cast<const Vec<T, V>*>(p); }
template <int BYTES> struct Raw;
template <> struct Raw<16> { typedef uint4 type; };
template <> struct Raw<8> { typedef uint2 type; };
template <> struct Raw<4> { typedef uint32_t type; };
template <> struct Raw<2> { typedef unsigned short type; };
template <typename T, int V> __device__ __forceinline__ Vec<T, V> load_last(const T* p) {
    typedef typename Raw<sizeof(T) * V>::type R;
    const R r = __ldcs(reinterpret_cast<const R*>(p));
    return *reinterpret_cast<const Vec<T, V>*>(&r);
}
template <typename T, int V> __device__ __forceinline__ void store_last(T* p, const Vec<T, V>& v) {
    typedef typename Raw<sizeof(T) * V>::type R;
    __stcs(reinterpret_cast<R*>(p), *reinterpret_cast<const R*>(&v));
}

// The logistic function by ex2 and reciprocal of the special-function unit: 2e-7 relative near zero and 6e-8 |u| far from
// it (the rounding of the exponent), where the product with u is off by at most 3e-8; u -> -inf gives 0.
__device__ __forceinline__ Two logistic(Two u) {
    float2 e = split(mul2(u, both(-1.44269504f)));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e.x));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e.y));
    e = split(add2(two(e.x, e.y), both(1.0f)));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(e.x));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(e.y));
    return two(e.x, e.y);
}
// twice the normal distribution function
__device__ __forceinline__ Two gauss2(Two u) {
    const float2 f = split(mul2(u, both(0.70710678f)));
    return add2(two(erff(f.x), erff(f.y)), both(1.0f));
}
template <int ACT> __device__ __forceinline__ Two act_value(Two u) {
    if (ACT == kActSilu) return mul2(u, logistic(u));
    if (ACT == kActGelu) return mul2(mul2(u, both(0.5f)), gauss2(u));
    return u;
}
// (__expf in GELU's slope: its error, 2 units of the last place and more for large arguments, is multiplied by a factor that
// falls off as fast: below 1e-7 of the slope's largest value.)
template <int ACT> __device__ __forceinline__ Two act_slope(Two u) {
    if (ACT == kActSilu) {
        const Two s = logistic(u);
        return mul2(s, fma2(u, fma2(s, both(-1.0f), both(1.0f)), both(1.0f)));
    }
    if (ACT == kActGelu) {
        const float2 f = split(mul2(mul2(u, u), both(-0.5f)));
        return fma2(mul2(u, both(0.39894228f)), two(__expf(f.x), __expf(f.y)), mul2(gauss2(u), both(0.5f)));
    }
    return both(1.0f);
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
    float* coef;                 // forward [B,C,2] k, q; backward [B,C,4] k, q, kx, kc: see the second passes
    int64_t elems;               // values of one image
    int64_t rows;                // rows of one image (the last may be short)
    int tiles, tile_rows, whole_tiles;   // of an image; whole_tiles: those in which every row is whole
    int64_t x_batch, x_row, dy_batch, dy_row, y_batch;   // strides in values
    int batch, chunks, C, G, cpg;
    int L, P;                    // values and vectors per row
    int first;                   // first image of this turn
    int wdtype, act;
    float eps, share;            // share: 1 / G, of a pixel's values that belong to one group
    float per_cpg;               // 1 / cpg: (c + 1/2) / cpg cut to an integer is c's group
};

// What a thread of the walk owns: vector `vec` of rows r0 + lane_row, step rows apart.
struct Walk {
    int rp, lane_row;            // rows the CTA takes at once, this thread's row among them
    bool on;
};
__device__ __forceinline__ Walk make_walk(const Args& a, int v0) {
    Walk w;
    if (a.P <= kThreads) {
        w.rp = kThreads / a.P;
        w.lane_row = threadIdx.x / a.P;
        w.on = w.lane_row < w.rp;
    } else {
        w.rp = 1;
        w.lane_row = 0;
        w.on = v0 + (int)threadIdx.x < a.P;
    }
    return w;
}

// An image's rows are cut into tiles of rp * unroll rows, and a CTA takes every chunks-th of them: at any time the whole
// grid reads one window of the image.  The second passes go through the tiles from the last to the first, the order in
// which L2 still holds them: of a 133 MB image half is found there.
__device__ __forceinline__ int tiles_of(const Args& a, int chunk) { return (a.tiles - 1 - chunk) / a.chunks + 1; }
// values of vector `vec` that row `row` has: V, or fewer at the image's end
template <int V> __device__ __forceinline__ int valid(const Args& a, int64_t row, int vec) {
    const int64_t left = a.elems - row * a.L - (int64_t)vec * V;
    return left >= V ? V : left > 0 ? (int)left : 0;
}
template <typename T, int V> __device__ __forceinline__ Vec<T, V> load_some(const T* p, int n) {
    Vec<T, V> v{};
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (j < n) v.v[j] = p[j];
    return v;
}
template <typename T, int V> __device__ __forceinline__ void store_some(T* p, const Vec<T, V>& v, int n) {
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (j < n) p[j] = v.v[j];
}

// ---- forward, pass 1: mean and centred square sum of every group over one chunk of one image ----------------------
// Squares are taken around the mean k of the thread's first rows: when k is far from the mean of the rest, the rows
// that k came from are themselves far from it and the variance is at least kUnroll/n of that distance squared, so
// the cancellation in q - s^2/n costs at most n/kUnroll units of the last place, whatever the mean.
// out(group, mean, m2) takes the result; sh: three floats for every entry.
template <typename T, int V, typename Out> __device__ __forceinline__ void chunk_stats(const Args& a, int b, int chunk, float* sh, Out out) {
    const T* x = static_cast<const T*>(a.x) + b * a.x_batch;
    const int slots = (a.P <= kThreads ? kThreads / a.P : 1) * a.L;   // entries of the CTA: [row][value of the row]
    float *s_n = sh, *s_mean = sh + slots, *s_m2 = sh + 2 * slots;
    for (int v0 = 0; v0 < a.P; v0 += kThreads) {
        const Walk w = make_walk(a, v0);
        if (!w.on) continue;
        const int vec = v0 + (a.P <= kThreads ? (int)threadIdx.x % a.P : (int)threadIdx.x);
        constexpr int H = (V + 1) / 2;
        const int64_t step = w.rp * a.x_row, next = (int64_t)a.chunks * a.tile_rows * a.x_row;
        const int64_t row0 = (int64_t)chunk * a.tile_rows + w.lane_row;
        const T* p = x + row0 * a.x_row + (int64_t)vec * V;
        Two minus[H], sum[H], square[H];   // minus: -k
#pragma unroll
        for (int i = 0; i < H; ++i) minus[i] = sum[i] = square[i] = both(0.0f);
        int got = 0;
        Vec<T, V> f[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (valid<V>(a, row0 + u * w.rp, vec) == V) {
                f[u] = load<T, V>(p + u * step);
                ++got;
            }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (u < got) {
#pragma unroll
                for (int i = 0; i < H; ++i) minus[i] = add2(minus[i], f[u].pair(i));
            }
#pragma unroll
        for (int i = 0; i < H; ++i) minus[i] = mul2(minus[i], both(-1.0f / max(got, 1)));
        auto add = [&](const Vec<T, V>& x) {
#pragma unroll
            for (int i = 0; i < H; ++i) {
                const Two d = add2(x.pair(i), minus[i]);
                sum[i] = add2(sum[i], d);
                square[i] = fma2(d, d, square[i]);
            }
        };
        int n = 0, tail = 0;        // rows, and values of the short row when it is this thread's
        const T* short_row = p;
        for (int i = tiles_of(a, chunk), tile = chunk; i > 0; --i, tile += a.chunks, p += next) {
            if (tile < a.whole_tiles) {
                Vec<T, V> v[kUnroll];
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) v[u] = load<T, V>(p + u * step);
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) add(v[u]);
                n += kUnroll;
            } else {
                for (int u = 0; u < kUnroll; ++u) {
                    const int has = valid<V>(a, (int64_t)tile * a.tile_rows + w.lane_row + u * w.rp, vec);
                    if (has == V) {
                        add(load<T, V>(p + u * step));
                        ++n;
                    } else if (has > 0) {
                        tail = has;
                        short_row = p + u * step;
                    }
                }
            }
        }
        float k[V], s[V], q[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float2 m = split(minus[j / 2]), t = split(sum[j / 2]), z = split(square[j / 2]);
            k[j] = j & 1 ? -m.y : -m.x;
            s[j] = j & 1 ? t.y : t.x;
            q[j] = j & 1 ? z.y : z.x;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            int nj = n;
            if (j < tail) {
                const float v = to_f(short_row[j]);
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
    // `lanes` threads join the entries of a group: first the mean, then the squares around it
    int lanes = 32;
    while (lanes > 1 && lanes * a.G > kThreads) lanes >>= 1;
    const int lane = threadIdx.x & (lanes - 1), pixels = slots / a.C;
    const int px0 = lane / a.cpg, ci0 = lane % a.cpg, dpx = lanes / a.cpg, dci = lanes % a.cpg;
    auto each = [&](int g, auto f) {
        for (int px = px0, ci = ci0; px < pixels;) {
            f(px * a.C + g * a.cpg + ci);
            px += dpx;
            ci += dci;
            if (ci >= a.cpg) {
                ci -= a.cpg;
                ++px;
            }
        }
    };
    auto lanes_sum = [&](float v) {
        for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
        return v;
    };
    for (int g0 = 0; g0 < a.G; g0 += kThreads / lanes) {
        const int g = min(g0 + (int)threadIdx.x / lanes, a.G - 1);   // (whole warps take part in the sums)
        const float near = s_mean[g * a.cpg];   // a value of the group's size: differences from it are added up
        float n = 0.0f, t = 0.0f, m2 = 0.0f;
        each(g, [&](int e) {
            n += s_n[e];
            if (s_n[e] > 0.0f) t = fmaf(s_n[e], s_mean[e] - near, t);
        });
        n = lanes_sum(n);
        t = lanes_sum(t);
        const float mean = n > 0.0f ? near + t / n : 0.0f;
        each(g, [&](int e) {
            if (s_n[e] > 0.0f) {
                const float d = s_mean[e] - mean;
                m2 += fmaf(s_n[e] * d, d, s_m2[e]);
            }
        });
        m2 = lanes_sum(m2);
        if (lane == 0 && g0 + (int)threadIdx.x / lanes < a.G) out(g, mean, m2);
    }
}
template <typename T, int V>
__global__ void __launch_bounds__(kThreads, kCtas) gn_stats_kernel(const Args a) {
    extern __shared__ float sh[];
    let_next_start();
    wait_for_previous();
    const int b = a.first + blockIdx.y, chunk = blockIdx.x;
    chunk_stats<T, V>(a, b, chunk, sh, [&](int g, float mean, float m2) {
        reinterpret_cast<float2*>(a.part)[((int64_t)b * a.G + g) * a.chunks + chunk] = make_float2(mean, m2);
    });
}

// values of one group in one chunk
__device__ __forceinline__ float chunk_count(const Args& a, int chunk) {
    const int n = tiles_of(a, chunk);
    int64_t e = (int64_t)n * a.tile_rows * a.L;
    if (chunk + (n - 1) * a.chunks == a.tiles - 1) e -= (int64_t)a.tiles * a.tile_rows * a.L - a.elems;   // the last tile
    return (float)e * a.share;
}

// u = k x + q of a channel; q is rounded at the size of mean rstd, as mean itself is
__device__ __forceinline__ float2 forward_coef(const Args& a, int ch, float2 st) {
    const float k = st.y * (a.weight ? load_param(a.weight, a.wdtype, ch) : 1.0f);
    return make_float2(k, fmaf(-st.x, k, a.bias ? load_param(a.bias, a.wdtype, ch) : 0.0f));
}
// and dx = k du + kx x + kc, with the group's means of w du and of w du xhat
__device__ __forceinline__ float4 backward_coef(const Args& a, int ch, float2 st, float m1, float m2) {
    const float2 f = forward_coef(a, ch, st);
    const float kx = -st.y * st.y * m2;
    return make_float4(f.x, f.y, kx, fmaf(-st.x, kx, -st.y * m1));
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
    const float total = (float)a.elems * a.share, near = part[0].x;
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
    const float rstd = 1.0f / sqrtf(m2 / total + a.eps);
    if (threadIdx.x == 0) reinterpret_cast<float2*>(a.stats)[bg] = make_float2(mean, rstd);
    const int first = (int)(bg % a.G) * a.cpg;
    for (int i = threadIdx.x; i < a.cpg; i += kJoinThreads)
        reinterpret_cast<float2*>(a.coef)[bg * a.cpg + i] = forward_coef(a, first + i, make_float2(mean, rstd));
}

// channel of value j of a vector
template <int V> __device__ __forceinline__ int channel(const Args& a, int vec, int j) {
    const int e = vec * V + (V == 1 ? 0 : j);
    return a.L == a.C ? e : e % a.C;
}

// ---- forward, pass 2 -----------------------------------------------------------------------------------------------
// c: k and q of the image's channels
template <typename T, int V, int ACT> __device__ __forceinline__ void chunk_apply(const Args& a, int b, int chunk, const float2* c) {
    const T* x = static_cast<const T*>(a.x) + b * a.x_batch;
    T* y = static_cast<T*>(a.y) + b * a.y_batch;
    for (int v0 = 0; v0 < a.P; v0 += kThreads) {
        const Walk w = make_walk(a, v0);
        if (!w.on) continue;
        const int vec = v0 + (a.P <= kThreads ? (int)threadIdx.x % a.P : (int)threadIdx.x);
        constexpr int H = (V + 1) / 2;
        Two k[H], q[H];
#pragma unroll
        for (int i = 0; i < H; ++i) {
            const float2 c0 = c[channel<V>(a, vec, 2 * i)], c1 = c[channel<V>(a, vec, 2 * i + 1)];
            k[i] = two(c0.x, c1.x);
            q[i] = two(c0.y, c1.y);
        }
        auto value = [&](const Vec<T, V>& v) {
            Vec<T, V> res;
#pragma unroll
            for (int i = 0; i < H; ++i) res.set(i, act_value<ACT>(fma2(v.pair(i), k[i], q[i])));
            return res;
        };
        const int64_t step = w.rp * a.x_row, ostep = (int64_t)w.rp * a.L;
        for (int tile = chunk + (tiles_of(a, chunk) - 1) * a.chunks; tile >= 0; tile -= a.chunks) {
            const int64_t row = (int64_t)tile * a.tile_rows + w.lane_row;
            const T* p = x + row * a.x_row + (int64_t)vec * V;
            T* o = y + row * a.L + (int64_t)vec * V;
            if (tile < a.whole_tiles) {
                Vec<T, V> v[kUnroll];
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) v[u] = load_last<T, V>(p + u * step);
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) store_last<T, V>(o + u * ostep, value(v[u]));
            } else {
                for (int u = 0; u < kUnroll; ++u) {
                    const int has = valid<V>(a, row + u * w.rp, vec);
                    if (has == V) store_last<T, V>(o + u * ostep, value(load_last<T, V>(p + u * step)));
                    else store_some<T, V>(o + u * ostep, value(load_some<T, V>(p + u * step, has)), has);
                }
            }
        }
    }
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads, kCtas) gn_apply_kernel(const Args a) {
    let_next_start();
    wait_for_previous();
    const int b = a.first + blockIdx.y;
    chunk_apply<T, V, ACT>(a, b, blockIdx.x, reinterpret_cast<const float2*>(a.coef) + (int64_t)b * a.C);
}

// ---- forward of a small image: both passes in one CTA ---------------------------------------------------------------
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads, kCtas) gn_small_kernel(const Args a) {
    extern __shared__ float sh[];   // k and q of every channel, mean and rstd of every group, entries
    let_next_start();
    wait_for_previous();
    const int b = blockIdx.x;
    float2* const coef = reinterpret_cast<float2*>(sh);
    float2* const stats = coef + a.C;
    const float total = (float)a.elems * a.share;
    chunk_stats<T, V>(a, b, 0, sh + 2 * (a.C + a.G), [&](int g, float mean, float m2) {
        const float2 st = make_float2(mean, 1.0f / sqrtf(m2 / total + a.eps));
        stats[g] = st;
        reinterpret_cast<float2*>(a.stats)[(int64_t)b * a.G + g] = st;
    });
    __syncthreads();
    for (int ch = threadIdx.x; ch < a.C; ch += kThreads) coef[ch] = forward_coef(a, ch, stats[ch / a.cpg]);
    __syncthreads();
    chunk_apply<T, V, ACT>(a, b, 0, coef);
}

// ---- backward, pass 1: sum of du and of du xhat per channel over one chunk ----------------------------------------
// out(channel, sums) takes the result; sh: two floats for every entry.
template <typename T, int V, int ACT, typename Out>
__device__ __forceinline__ void chunk_grad_sums(const Args& a, int b, int chunk, float* sh, Out out) {
    const T* x = static_cast<const T*>(a.x) + b * a.x_batch;
    const T* dy = static_cast<const T*>(a.dy) + b * a.dy_batch;
    const int slots = (a.P <= kThreads ? kThreads / a.P : 1) * a.L;
    float *s_1 = sh, *s_2 = sh + slots;
    for (int v0 = 0; v0 < a.P; v0 += kThreads) {
        const Walk w = make_walk(a, v0);
        if (!w.on) continue;
        const int vec = v0 + (a.P <= kThreads ? (int)threadIdx.x % a.P : (int)threadIdx.x);
        constexpr int H = (V + 1) / 2;
        Two minus[H], k[H], q[H], s1[H], s2[H];   // u = k (x - mean) + q; s2 sums du (x - mean)
        float rstd[V];
#pragma unroll
        for (int i = 0; i < H; ++i) {
            float2 st[2];
            float wt[2], bs[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int ch = channel<V>(a, vec, 2 * i + j);
                st[j] = reinterpret_cast<const float2*>(a.stats)[(int64_t)b * a.G + (int)(((float)ch + 0.5f) * a.per_cpg)];
                wt[j] = a.weight ? load_param(a.weight, a.wdtype, ch) : 1.0f;
                bs[j] = a.bias ? load_param(a.bias, a.wdtype, ch) : 0.0f;
                if (2 * i + j < V) rstd[2 * i + j] = st[j].y;
            }
            minus[i] = two(-st[0].x, -st[1].x);
            k[i] = two(st[0].y * wt[0], st[1].y * wt[1]);
            q[i] = two(bs[0], bs[1]);
            s1[i] = s2[i] = both(0.0f);
        }
        auto add = [&](const Vec<T, V>& x, const Vec<T, V>& dy) {
#pragma unroll
            for (int i = 0; i < H; ++i) {
                const Two d = add2(x.pair(i), minus[i]);
                const Two du = mul2(dy.pair(i), act_slope<ACT>(fma2(d, k[i], q[i])));
                s1[i] = add2(s1[i], du);
                s2[i] = fma2(du, d, s2[i]);
            }
        };
        const int64_t step = w.rp * a.x_row, dstep = w.rp * a.dy_row;
        for (int i = tiles_of(a, chunk), tile = chunk; i > 0; --i, tile += a.chunks) {
            const int64_t row = (int64_t)tile * a.tile_rows + w.lane_row;
            const T* p = x + row * a.x_row + (int64_t)vec * V;
            const T* d = dy + row * a.dy_row + (int64_t)vec * V;
            if (tile < a.whole_tiles) {
                Vec<T, V> v[kUnroll2], g[kUnroll2];
#pragma unroll
                for (int u = 0; u < kUnroll2; ++u) {
                    v[u] = load<T, V>(p + u * step);
                    g[u] = load<T, V>(d + u * dstep);
                }
#pragma unroll
                for (int u = 0; u < kUnroll2; ++u) add(v[u], g[u]);
            } else {
                for (int u = 0; u < kUnroll2; ++u) {   // dy of zero behind the image's end
                    const int has = valid<V>(a, row + u * w.rp, vec);
                    if (has > 0) add(load_some<T, V>(p + u * step, has), load_some<T, V>(d + u * dstep, has));
                }
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float2 t1 = split(s1[j / 2]), t2 = split(s2[j / 2]);
            s_1[w.lane_row * a.L + vec * V + j] = j & 1 ? t1.y : t1.x;
            s_2[w.lane_row * a.L + vec * V + j] = (j & 1 ? t2.y : t2.x) * rstd[j];
        }
    }
    __syncthreads();
    for (int ch = threadIdx.x; ch < a.C; ch += kThreads) {
        float t1 = 0.0f, t2 = 0.0f;
        for (int e = ch; e < slots; e += a.C) {
            t1 += s_1[e];
            t2 += s_2[e];
        }
        out(ch, make_float2(t1, t2));
    }
}
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads, kCtas2) gn_grad_sums_kernel(const Args a) {
    extern __shared__ float sh[];
    let_next_start();
    wait_for_previous();
    const int b = a.first + blockIdx.y, chunk = blockIdx.x;
    float2* const part = reinterpret_cast<float2*>(a.part) + ((int64_t)b * a.chunks + chunk) * a.C;
    chunk_grad_sums<T, V, ACT>(a, b, chunk, sh, [&](int ch, float2 t) { part[ch] = t; });
}

// ---- backward, join: one CTA per (image, group): the sums of its channels over the chunks, the group's means, and the
// coefficients of the second pass ---------------------------------------------------------------------------------------
__global__ void __launch_bounds__(kJoinThreads) gn_grad_join_kernel(const Args a) {
    __shared__ float2 sh[kJoinThreads];
    __shared__ float sw[2][kJoinThreads / 32];
    let_next_start();
    wait_for_previous();
    const int g = blockIdx.x, b = a.first + blockIdx.y, first = g * a.cpg;
    const int wide = min(a.cpg, kJoinThreads), parts = kJoinThreads / wide;   // channels at once, threads of each
    const int in = threadIdx.x % wide, part = threadIdx.x / wide;
    int top = 1;
    while (top < parts) top <<= 1;
    float2* sums = reinterpret_cast<float2*>(a.sums) + (int64_t)b * a.C + first;
    float m1 = 0.0f, m2 = 0.0f;
    for (int c0 = 0; c0 < a.cpg; c0 += wide) {
        const int i = c0 + in;
        float2 t = make_float2(0.0f, 0.0f);
        if (i < a.cpg && part < parts) {
            const float2* p = reinterpret_cast<const float2*>(a.part) + (int64_t)b * a.chunks * a.C + first + i;
#pragma unroll 4
            for (int k = part; k < a.chunks; k += parts) {
                const float2 v = p[(int64_t)k * a.C];
                t.x += v.x;
                t.y += v.y;
            }
        }
        sh[threadIdx.x] = t;
        __syncthreads();
        for (int half = top >> 1; half > 0; half >>= 1) {
            if (part < half && part + half < parts) {
                sh[threadIdx.x].x += sh[threadIdx.x + half * wide].x;
                sh[threadIdx.x].y += sh[threadIdx.x + half * wide].y;
            }
            __syncthreads();
        }
        if (part == 0 && i < a.cpg) {
            t = sh[threadIdx.x];
            sums[i] = t;
            const float w = a.weight ? load_param(a.weight, a.wdtype, first + i) : 1.0f;
            m1 = fmaf(w, t.x, m1);
            m2 = fmaf(w, t.y, m2);
        }
        __syncthreads();
    }
    const float inv = 1.0f / ((float)a.elems * a.share);
    m1 = cta_sum(m1, sw[0]) * inv;
    m2 = cta_sum(m2, sw[1]) * inv;
    const float2 st = reinterpret_cast<const float2*>(a.stats)[(int64_t)b * a.G + g];
    for (int i = threadIdx.x; i < a.cpg; i += kJoinThreads)
        reinterpret_cast<float4*>(a.coef)[(int64_t)b * a.C + first + i] = backward_coef(a, first + i, st, m1, m2);
}

// ---- backward, pass 2: dx, and (last turn) the parameter gradients ------------------------------------------------
// the parameter gradients of channel ch: over all images
__device__ __forceinline__ void param_grads(const Args& a, int ch) {
    const float2* sums = reinterpret_cast<const float2*>(a.sums) + ch;
    float t1 = 0.0f, t2 = 0.0f;
    for (int k = 0; k < a.batch; ++k) {
        const float2 s = sums[(int64_t)k * a.C];
        t1 += s.x;
        t2 += s.y;
    }
    if (a.dweight) store_param(a.dweight, a.wdtype, ch, t2);
    if (a.dbias) store_param(a.dbias, a.wdtype, ch, t1);
}
template <typename T, int V, int ACT> __device__ __forceinline__ void chunk_grad_apply(const Args& a, int b, int chunk, const float4* c) {
    const T* x = static_cast<const T*>(a.x) + b * a.x_batch;
    const T* dy = static_cast<const T*>(a.dy) + b * a.dy_batch;
    T* dx = static_cast<T*>(a.y) + b * a.y_batch;
    for (int v0 = 0; v0 < a.P; v0 += kThreads) {
        const Walk w = make_walk(a, v0);
        if (!w.on) continue;
        const int vec = v0 + (a.P <= kThreads ? (int)threadIdx.x % a.P : (int)threadIdx.x);
        constexpr int H = (V + 1) / 2;
        Two k[H], q[H], kx[H], kc[H];
#pragma unroll
        for (int i = 0; i < H; ++i) {
            const float4 c0 = c[channel<V>(a, vec, 2 * i)], c1 = c[channel<V>(a, vec, 2 * i + 1)];
            k[i] = two(c0.x, c1.x);
            q[i] = two(c0.y, c1.y);
            kx[i] = two(c0.z, c1.z);
            kc[i] = two(c0.w, c1.w);
        }
        auto value = [&](const Vec<T, V>& x, const Vec<T, V>& dy) {
            Vec<T, V> res;
#pragma unroll
            for (int i = 0; i < H; ++i) {
                const Two v = x.pair(i), du = mul2(dy.pair(i), act_slope<ACT>(fma2(v, k[i], q[i])));
                res.set(i, fma2(k[i], du, fma2(kx[i], v, kc[i])));
            }
            return res;
        };
        const int64_t step = w.rp * a.x_row, dstep = w.rp * a.dy_row, ostep = (int64_t)w.rp * a.L;
        for (int tile = chunk + (tiles_of(a, chunk) - 1) * a.chunks; tile >= 0; tile -= a.chunks) {
            const int64_t row = (int64_t)tile * a.tile_rows + w.lane_row;
            const T* p = x + row * a.x_row + (int64_t)vec * V;
            const T* d = dy + row * a.dy_row + (int64_t)vec * V;
            T* o = dx + row * a.L + (int64_t)vec * V;
            if (tile < a.whole_tiles) {
                Vec<T, V> v[kUnroll2], g[kUnroll2];
#pragma unroll
                for (int u = 0; u < kUnroll2; ++u) {
                    v[u] = load_last<T, V>(p + u * step);
                    g[u] = load_last<T, V>(d + u * dstep);
                }
#pragma unroll
                for (int u = 0; u < kUnroll2; ++u) store_last<T, V>(o + u * ostep, value(v[u], g[u]));
            } else {
                for (int u = 0; u < kUnroll2; ++u) {
                    const int has = valid<V>(a, row + u * w.rp, vec);
                    if (has > 0)
                        store_some<T, V>(o + u * ostep, value(load_some<T, V>(p + u * step, has), load_some<T, V>(d + u * dstep, has)), has);
                }
            }
        }
    }
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads, kCtas2) gn_grad_apply_kernel(const Args a, int params) {
    let_next_start();
    wait_for_previous();
    const int b = a.first + blockIdx.y;
    if (params && blockIdx.y == 0)   // every CTA of one image takes a share of the channels
        for (int ch = blockIdx.x * kThreads + threadIdx.x; ch < a.C; ch += gridDim.x * kThreads) param_grads(a, ch);
    if (a.y) chunk_grad_apply<T, V, ACT>(a, b, blockIdx.x, reinterpret_cast<const float4*>(a.coef) + (int64_t)b * a.C);
}

// ---- backward of a small image: both passes in one CTA; the parameter gradients of several images in another launch ---
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads, kCtas2) gn_small_grad_kernel(const Args a) {
    extern __shared__ float4 sh4[];   // coefficients of every channel, its sums, means of every group, entries
    let_next_start();
    wait_for_previous();
    const int b = blockIdx.x;
    float4* const coef = sh4;
    float2* const sums = reinterpret_cast<float2*>(coef + a.C);
    float2* const means = sums + a.C;
    chunk_grad_sums<T, V, ACT>(a, b, 0, reinterpret_cast<float*>(means + a.G), [&](int ch, float2 t) {
        sums[ch] = t;
        reinterpret_cast<float2*>(a.sums)[(int64_t)b * a.C + ch] = t;
        if (a.batch == 1) {
            if (a.dweight) store_param(a.dweight, a.wdtype, ch, t.y);
            if (a.dbias) store_param(a.dbias, a.wdtype, ch, t.x);
        }
    });
    if (!a.y) return;
    __syncthreads();
    const float inv = 1.0f / ((float)a.elems * a.share);
    for (int g = threadIdx.x >> 5; g < a.G; g += kThreads / 32) {
        float m1 = 0.0f, m2 = 0.0f;
        for (int i = threadIdx.x & 31; i < a.cpg; i += 32) {
            const int ch = g * a.cpg + i;
            const float w = a.weight ? load_param(a.weight, a.wdtype, ch) : 1.0f;
            m1 = fmaf(w, sums[ch].x, m1);
            m2 = fmaf(w, sums[ch].y, m2);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            m1 += __shfl_xor_sync(~0u, m1, o);
            m2 += __shfl_xor_sync(~0u, m2, o);
        }
        if ((threadIdx.x & 31) == 0) means[g] = make_float2(m1 * inv, m2 * inv);
    }
    __syncthreads();
    for (int ch = threadIdx.x; ch < a.C; ch += kThreads) {
        const int g = ch / a.cpg;
        coef[ch] = backward_coef(a, ch, reinterpret_cast<const float2*>(a.stats)[(int64_t)b * a.G + g], means[g].x, means[g].y);
    }
    __syncthreads();
    chunk_grad_apply<T, V, ACT>(a, b, 0, coef);
}
__global__ void __launch_bounds__(kThreads) gn_params_kernel(const Args a) {
    let_next_start();
    wait_for_previous();
    const int ch = blockIdx.x * kThreads + threadIdx.x;
    if (ch < a.C) param_grads(a, ch);
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

// Images per turn: as many as keep the turn's inputs within kTurnBytes, at least one, and the turns about equal.
int images_per_turn(const D3gsGroupNorm& d, bool backward) {
    const int64_t image = d.pixels * d.channels * elem_size(d.dtype) * (backward ? 2 : 1);
    int64_t n = kTurnBytes / (image > 0 ? image : 1);
    if (n < 1) n = 1;
    return d.batch ? (int)div_up64(d.batch, div_up64(d.batch, n)) : 1;
}

// An image by one CTA, both passes in one launch (the backward of a batch takes one more), or every image by many CTAs
// with a join between the passes: one CTA is slower with the image, a launch is not.  Measured with 64 channels, many
// CTAs -> one, us: forward of a float32 image of 16 KB 15 -> 12, 64 KB 15 -> 12, 128 KB 15 -> 15 (bf16 17 -> 18), 256 KB
// 16 -> 19; backward 16 KB 13 -> 10, 32 KB 13 -> 10 (16 images of bf16 17 -> 17), 64 KB 13 -> 12 (bf16 17 -> 18, 16
// images 17 -> 22), 128 KB 13 -> 17.  Where there is an image for every SM one CTA also finds its image in L2 again:
// 200 images of 16 KB 22 -> 14 and 24 -> 22, of 512 KB 80 -> 59 and 130 -> 110.  (Many channels would leave a CTA no
// shared memory for their coefficients.)
constexpr int kSmallChannels = 2048;
bool one_cta(const D3gsGroupNorm& d, const Args& a, bool backward) {
    const int64_t vectors = a.elems / (a.L / a.P);   // what a thread loads at a time, 16 bytes in the figures above
    return d.channels <= kSmallChannels && vectors <= (d.batch >= 148 ? kSmallMany : backward ? kSmallGrad : kSmall);
}

// Chunks of one image: as many CTAs in a turn as run at once (a CTA without a tile is not launched).
int chunks_of(const D3gsGroupNorm& d, bool backward) {
    const int64_t n = div_up64((backward ? kCtas2 : kCtas) * 148, images_per_turn(d, backward));
    return (int)(n > kMaxChunks ? kMaxChunks : n);
}

int32_t check(const D3gsGroupNorm* d, const char* what) {
    D3GS_REQUIRE(d != nullptr, "%s: desc is NULL", what);
    D3GS_REQUIRE(d->batch >= 0 && d->batch <= 65535 && d->pixels >= 0, "%s: batch %lld (at most 65535), pixels %lld", what,
                 (long long)d->batch, (long long)d->pixels);
    D3GS_REQUIRE(d->channels >= 1 && d->channels <= kMaxChannels, "%s: %d channels (1 to %d)", what, d->channels, kMaxChannels);
    D3GS_REQUIRE(d->groups >= 1 && d->channels % d->groups == 0, "%s: %d groups do not divide %d channels", what, d->groups,
                 d->channels);
    D3GS_REQUIRE(d->pixels < (int64_t)1 << 31, "%s: image too large", what);
    D3GS_REQUIRE(d->dtype >= 0 && d->dtype <= 2 && d->weight_dtype >= 0 && d->weight_dtype <= 2, "%s: dtype %d / %d", what,
                 d->dtype, d->weight_dtype);
    D3GS_REQUIRE(d->act >= 0 && d->act <= 2, "%s: act %d", what, d->act);
    D3GS_REQUIRE(d->x_batch_stride >= 0 && d->x_pixel_stride >= 0 && d->dy_batch_stride >= 0 && d->dy_pixel_stride >= 0,
                 "%s: strides must not be negative", what);
    D3GS_REQUIRE(d->eps >= 0.0f, "%s: eps must not be negative", what);
    return D3GS_OK;
}

struct Workspace {
    size_t sums, coef, bytes;   // offsets (the partial sums come first), total
};
Workspace workspace_of(const D3gsGroupNorm& d, bool backward) {
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    Workspace w;
    const size_t chunks = chunks_of(d, backward), channels = (size_t)d.batch * d.channels;
    w.sums = up((size_t)d.batch * chunks * (backward ? d.channels : d.groups) * 8);
    w.coef = w.sums + (backward ? up(channels * 8) : 0);
    w.bytes = w.coef + up(channels * (backward ? 16 : 8)) + 256;
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
    a.tile_rows = (a.P <= kThreads ? kThreads / a.P : 1) * (backward ? kUnroll2 : kUnroll);
    a.tiles = (int)div_up64(a.rows, a.tile_rows);
    a.whole_tiles = (int)(a.elems / ((int64_t)a.tile_rows * a.L));
    if (a.chunks > a.tiles) a.chunks = a.tiles;        // no empty chunk
    a.x_batch = d.x_batch_stride;
    a.dy_batch = d.dy_batch_stride;
    a.x_row = a.L == a.C ? d.x_pixel_stride : a.L;
    a.dy_row = a.L == a.C ? d.dy_pixel_stride : a.L;
    a.y_batch = a.elems;
    a.batch = (int)d.batch;
    a.wdtype = d.weight_dtype;
    a.act = d.act;
    a.eps = d.eps;
    a.share = 1.0f / d.groups;
    a.per_cpg = 1.0f / a.cpg;
    a.part = static_cast<float*>(ws);
    a.coef = reinterpret_cast<float*>(static_cast<char*>(ws) + w.coef);
    a.sums = reinterpret_cast<float*>(static_cast<char*>(ws) + w.sums);
    return a;
}

// most: the most dynamic shared memory that any call of this kernel asks for.  The attribute belongs to the kernel, not to
// the call: set to what a call needs, another thread's smaller call could lower it between this one's two steps.
template <typename K, typename... A>
int32_t launch(K kernel, const char* name, dim3 grid, unsigned threads, size_t smem, size_t most, cudaStream_t st, const A&... args) {
    if (smem > 48 * 1024) D3GS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
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

// Dynamic shared memory: entries (values of the rows that a CTA takes at once), per-channel and per-group values.
size_t entries(const Args& a) { return (size_t)(a.P <= kThreads ? kThreads / a.P : 1) * a.L; }
constexpr size_t most_entries(int V, int channels) { return channels > kThreads * V ? channels : kThreads * V; }
constexpr size_t small_bytes(size_t entries, size_t c, size_t g) { return entries * 12 + (c + g) * 8; }
constexpr size_t small_grad_bytes(size_t entries, size_t c, size_t g) { return entries * 8 + c * 24 + g * 8; }

template <typename T, int V, int ACT>
int32_t run_forward(const D3gsGroupNorm& d, Args a, cudaStream_t st) {
    const int turn = images_per_turn(d, false);
    const size_t slots = entries(a);
    if (one_cta(d, a, false)) {
        a.chunks = 1;
        return launch(gn_small_kernel<T, V, ACT>, "gn_small_kernel", dim3(a.batch), kThreads, small_bytes(slots, a.C, a.G),
                      small_bytes(most_entries(V, kSmallChannels), kSmallChannels, kSmallChannels), st, a);
    }
    for (int b = 0; b < a.batch; b += turn) {
        const int images = b + turn <= a.batch ? turn : a.batch - b;
        a.first = b;
        const dim3 grid(a.chunks, images);
        if (int32_t rc = launch(gn_stats_kernel<T, V>, "gn_stats_kernel", grid, kThreads, slots * 12,
                                most_entries(V, kMaxChannels) * 12, st, a))
            return rc;
        if (int32_t rc = launch(gn_stats_join_kernel, "gn_stats_join_kernel", dim3(images * a.G), kJoinThreads, 0, 0, st, a)) return rc;
        if (int32_t rc = launch(gn_apply_kernel<T, V, ACT>, "gn_apply_kernel", grid, kThreads, 0, 0, st, a)) return rc;
    }
    return D3GS_OK;
}

template <typename T, int V, int ACT>
int32_t run_backward(const D3gsGroupNorm& d, Args a, cudaStream_t st) {
    const int turn = images_per_turn(d, true);
    const size_t slots = entries(a);
    if (one_cta(d, a, true)) {
        a.chunks = 1;
        if (int32_t rc = launch(gn_small_grad_kernel<T, V, ACT>, "gn_small_grad_kernel", dim3(a.batch), kThreads,
                                small_grad_bytes(slots, a.C, a.G),
                                small_grad_bytes(most_entries(V, kSmallChannels), kSmallChannels, kSmallChannels), st, a))
            return rc;
        if (a.batch == 1 || !(a.dweight || a.dbias)) return D3GS_OK;
        return launch(gn_params_kernel, "gn_params_kernel", dim3((a.C + kThreads - 1) / kThreads), kThreads, 0, 0, st, a);
    }
    for (int b = 0; b < a.batch; b += turn) {
        const int images = b + turn <= a.batch ? turn : a.batch - b;
        a.first = b;
        const dim3 grid(a.chunks, images);
        if (int32_t rc = launch(gn_grad_sums_kernel<T, V, ACT>, "gn_grad_sums_kernel", grid, kThreads, slots * 8,
                                most_entries(V, kMaxChannels) * 8, st, a))
            return rc;
        if (int32_t rc = launch(gn_grad_join_kernel, "gn_grad_join_kernel", dim3(a.G, images), kJoinThreads, 0, 0, st, a)) return rc;
        const int params = b + images == a.batch && (a.dweight || a.dbias);
        if (int32_t rc = launch(gn_grad_apply_kernel<T, V, ACT>, "gn_grad_apply_kernel", grid, kThreads, 0, 0, st, a, params))
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

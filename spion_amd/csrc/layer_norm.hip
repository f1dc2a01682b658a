// Layer norm of rows with the residual's addition ahead of it (the reference's layer adds in one operation and has nn.LayerNorm as the
// next, models/model_transformer.py:55-102) and its backward:
//   h = x + residual, rounded to the tensors' type: the stream as it goes on
//   mu = mean(h),  s = 1 / sqrt(mean((h - mu)^2) + eps),  xh = (h - mu) s,  y = xh w + b
//   g = dy w,  dh = s (g - mean(g) - xh mean(g xh)) + (gradient of the stream);   dw, db = sums over the rows of dy xh and dy
// Bound by memory: every tensor is read or written once.  A row lies in the registers of 8, 16, 64, 256 or 1024 lanes in pieces of 16
// bytes, so the mean, and the variance as the mean of squares about it (not as a difference of sums, which loses what a large mean leaves),
// need no second pass over memory.  Rows need not start on 16 bytes: the hardware loads and stores 16 bytes from any element's address, and
// only what is left of a row behind its last whole piece goes element by element.  The backward forms mu and s again (8 bytes a row
// less to keep) in two reductions of two sums each.  Rows longer than the registers are read again for each step (from L2).  Statistics
// and sums are fp32.  Work-groups walk several rows each: the weight is read once, and the backward leaves one partial dw and db a
// work-group, which a second launch adds up in a fixed order.  With a residual, us (bytes moved to the time, TB/s): 262144 x 64 fp32 forward 44
// (6.1, part of it from the cache), backward 44 + 4 for dw and db; 8192 x 4096 bf16 46 (5.8) and 58 to 61 + 9; 16384 x 1001 bf16, forward alone,
// 15 to 17 (3.9 to 4.3); one row of 768 3, the launch.
#include "common.h"
#include "tile_ops.h"
#include "../../include/spion_hip.h"

#include <algorithm>
#include <climits>

namespace spion {

struct LayerNormCall {
    const void *x, *res, *w, *b, *dy, *dh;
    void *y, *h, *dx;
    float* part;
    long long rows, xs, rs, dys, dhs;  // strides of rows, in elements; outputs are contiguous
    int n;
    float eps;
};

typedef unsigned words4 __attribute__((ext_vector_type(4)));
typedef unsigned words2 __attribute__((ext_vector_type(2)));
// (global memory instructions take any address here)
typedef words4 words4_anywhere __attribute__((aligned(2)));
typedef words2 words2_anywhere __attribute__((aligned(2)));
typedef unsigned word_anywhere __attribute__((aligned(2)));

// Elements i .. i + V - 1 of a row of n, those behind its end zeros: the words as they come from memory, so that nothing waits for them
// before all of a row's pieces are asked for, and then as floats.  (Converted where they are loaded, each piece waited for its own: backward
// of 8192 x 4096 bf16 107 us against 60.)
template <class T>
struct RowWords {
    static constexpr int V = 16 / sizeof(T);
    words4 u;
    // as if they had changed: what was made of them before is not kept for what follows
    __device__ __forceinline__ void again() {
        if constexpr (sizeof(T) == 2) asm volatile("" : "+v"(u));
    }
    // The row's last V where there are fewer from i on (one load for every lane), which down() then moves to where they belong.  It stands
    // apart, behind all loads, and rows of fewer than V elements (TINY) have kernels of their own: beside each load, either makes the
    // compiler wait for one before the next (262144 x 64 fp32, training: 92 and 104 us).
    template <bool TINY>
    __device__ __forceinline__ void load(const T* row, int i, int n) {
        u = words4{0, 0, 0, 0};
        if (i >= n) return;
        if constexpr (!TINY) {
            u = *reinterpret_cast<const words4_anywhere*>(row + min(i, n - V));
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (i + e < n) u[e] = reinterpret_cast<const unsigned*>(row)[i + e];
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (i + e < n) u[e / 2] |= (unsigned)reinterpret_cast<const unsigned short*>(row)[i + e] << (16 * (e & 1));
        }
    }
    __device__ __forceinline__ void down(int i, int n) {
        const int off = i - min(i, n - V);
        if (i >= n) return;
        if constexpr (sizeof(T) == 4) {
            if (off & 1) u = words4{u[1], u[2], u[3], 0};
            if (off & 2) u = words4{u[2], u[3], 0, 0};
        } else {
            if (off & 1) u = words4{u[0] >> 16 | u[1] << 16, u[1] >> 16 | u[2] << 16, u[2] >> 16 | u[3] << 16, u[3] >> 16};
            if (off & 2) u = words4{u[1], u[2], u[3], 0};
            if (off & 4) u = words4{u[2], u[3], 0, 0};
        }
    }
};
template <class T>
struct RowPiece {
    static constexpr int V = 16 / sizeof(T);
    float x[V];
    RowPiece() = default;
    __device__ __forceinline__ explicit RowPiece(const RowWords<T>& w) { take(w); }
    __device__ __forceinline__ void take(const RowWords<T>& w) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const unsigned bits = w.u[k];  // (a bit cast of a vector's element takes its first one)
            if constexpr (sizeof(T) == 4) {
                x[k] = __builtin_bit_cast(float, bits);
            } else {
                x[2 * k] = bf16_lo(bits);
                x[2 * k + 1] = bf16_hi(bits);
            }
        }
    }
    __device__ __forceinline__ void load(const T* row, int i, int n) {
        RowWords<T> w;
        w.template load<false>(row, i, n);
        if (n % V) w.down(i, n);
        take(w);
    }
    __device__ __forceinline__ void store(T* row, int i, int n) const {
        words4 u;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (sizeof(T) == 4) u[k] = __builtin_bit_cast(unsigned, x[k]);
            else u[k] = pack_bf16(x[2 * k], x[2 * k + 1]);
        }
        T* p = row + i;
        if (i + V <= n) {
            *reinterpret_cast<words4_anywhere*>(p) = u;
        } else if (i < n) {  // four, two and one of what is left
            const int left = n - i;
            if constexpr (sizeof(T) == 2) {
                if (left & 4) {
                    *reinterpret_cast<words2_anywhere*>(p) = words2{u[0], u[1]};
                    u = words4{u[2], u[3], 0, 0};
                    p += 4;
                }
                if (left & 2) {
                    *reinterpret_cast<word_anywhere*>(p) = u[0];
                    u[0] = u[1];
                    p += 2;
                }
                if (left & 1) *reinterpret_cast<unsigned short*>(p) = (unsigned short)u[0];
            } else {
                if (left & 2) {
                    *reinterpret_cast<words2_anywhere*>(p) = words2{u[0], u[1]};
                    u[0] = u[2];
                    p += 2;
                }
                if (left & 1) *reinterpret_cast<unsigned*>(p) = u[0];
            }
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = 0.f;
    }
};

// Two sums over the LANES lanes of a row.  More than a wavefront: through LDS, two sets of slots taken in turn so that one barrier
// a reduction is enough.
template <int LANES>
struct RowSums {
    float (*slots)[2][16];  // [2] sets
    int turn = 0;
    __device__ __forceinline__ void over(float& a, float& b) {
#pragma unroll
        for (int o = 1; o < (LANES < 64 ? LANES : 64); o <<= 1) {
            a += __shfl_xor(a, o, 64);
            b += __shfl_xor(b, o, 64);
        }
        if constexpr (LANES > 64) {
            float(*s)[16] = slots[turn];
            turn ^= 1;
            if ((threadIdx.x & 63) == 0) {
                s[0][threadIdx.x >> 6] = a;
                s[1][threadIdx.x >> 6] = b;
            }
            __syncthreads();
            a = s[0][0];
            b = s[1][0];
#pragma unroll
            for (int i = 1; i < LANES / 64; ++i) {
                a += s[0][i];
                b += s[1][i];
            }
        }
    }
    __device__ __forceinline__ float over(float a) {
        float none = 0.f;
        over(a, none);
        return a;
    }
};

// LANES lanes to a row of up to LANES * C * V elements; LANES <= 256: work-groups of 256 threads with 256 / LANES rows at a time.
template <int LANES>
constexpr int row_threads() { return LANES < 256 ? 256 : LANES; }

template <class T, int LANES, int C, bool TINY>
__global__ __launch_bounds__(row_threads<LANES>()) void layer_norm_forward_kernel(LayerNormCall a) {
    constexpr int V = RowPiece<T>::V, ROWS = row_threads<LANES>() / LANES;
    __shared__ float slots[2][2][16];
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    RowSums<LANES> sums{slots};
    RowWords<T> w[C], b[C];  // (words: converted where they are used)
#pragma unroll
    for (int c = 0; c < C; ++c) {
        w[c].template load<TINY>(reinterpret_cast<const T*>(a.w), (c * LANES + lane) * V, a.n);
        b[c].template load<TINY>(reinterpret_cast<const T*>(a.b), (c * LANES + lane) * V, a.b ? a.n : 0);
    }
    const bool whole = TINY || a.n % V == 0;
    if (!whole)
#pragma unroll
        for (int c = 0; c < C; ++c) {
            w[c].down((c * LANES + lane) * V, a.n);
            if (a.b) b[c].down((c * LANES + lane) * V, a.n);
        }
    const float rn = 1.f / a.n;
    for (long long r0 = (long long)blockIdx.x * ROWS; r0 < a.rows; r0 += (long long)gridDim.x * ROWS) {
        const long long row = r0 + sub;
        const int n = row < a.rows ? a.n : 0;
        RowPiece<T> h[C];
        RowWords<T> x[C], r[C];
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) x[c].template load<TINY>(reinterpret_cast<const T*>(a.x) + row * a.xs, (c * LANES + lane) * V, n);
        if (a.res)
#pragma unroll
            for (int c = 0; c < C; ++c) r[c].template load<TINY>(reinterpret_cast<const T*>(a.res) + row * a.rs, (c * LANES + lane) * V, n);
        if (!whole)
#pragma unroll
            for (int c = 0; c < C; ++c) {
                x[c].down((c * LANES + lane) * V, n);
                if (a.res) r[c].down((c * LANES + lane) * V, n);
            }
#pragma unroll
        for (int c = 0; c < C; ++c) h[c].take(x[c]);
        if (a.res) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                RowPiece<T> o;
                o.take(r[c]);
#pragma unroll
                for (int e = 0; e < V; ++e) h[c].x[e] = (float)(T)(h[c].x[e] + o.x[e]);
                h[c].store(reinterpret_cast<T*>(a.h) + row * a.n, (c * LANES + lane) * V, n);
            }
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) s += h[c].x[e];
        const float mu = sums.over(s) * rn;
        float q = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                h[c].x[e] -= mu;
                if ((c * LANES + lane) * V + e < a.n) q = fmaf(h[c].x[e], h[c].x[e], q);
            }
        const float inv = rsqrtf(sums.over(q) * rn + a.eps);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            w[c].again();
            b[c].again();
            const RowPiece<T> by(w[c]), to(b[c]);
#pragma unroll
            for (int e = 0; e < V; ++e) h[c].x[e] = fmaf(h[c].x[e] * inv, by.x[e], to.x[e]);
            h[c].store(reinterpret_cast<T*>(a.y) + row * a.n, (c * LANES + lane) * V, n);
        }
    }
}

// a.x is the stream h.  part: [work-groups][dw, db][n].
template <class T, int LANES, int C, bool TINY>
__global__ __launch_bounds__(row_threads<LANES>()) void layer_norm_backward_kernel(LayerNormCall a) {
    constexpr int V = RowPiece<T>::V, ROWS = row_threads<LANES>() / LANES, WIDTH = LANES * C * V;
    __shared__ float slots[2][2][16];
    __shared__ float folded[ROWS > 1 ? ROWS * WIDTH : 1];
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    RowSums<LANES> sums{slots};
    // Pieces stay words and are converted in each of the three steps: half the registers of bf16 rows, and twice the wavefronts.
    RowWords<T> w[C];
    float dw[C][V], db[C][V];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        w[c].template load<TINY>(reinterpret_cast<const T*>(a.w), (c * LANES + lane) * V, a.n);
        if (!TINY && a.n % V) w[c].down((c * LANES + lane) * V, a.n);
#pragma unroll
        for (int e = 0; e < V; ++e) dw[c][e] = db[c][e] = 0.f;
    }
    const bool whole = TINY || a.n % V == 0;
    const float rn = 1.f / a.n;
    for (long long r0 = (long long)blockIdx.x * ROWS; r0 < a.rows; r0 += (long long)gridDim.x * ROWS) {
        const long long row = r0 + sub;
        const int n = row < a.rows ? a.n : 0;
        RowWords<T> h[C], g[C], dh[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = (c * LANES + lane) * V;
            h[c].template load<TINY>(reinterpret_cast<const T*>(a.x) + row * a.xs, i, n);
            g[c].template load<TINY>(reinterpret_cast<const T*>(a.dy) + row * a.dys, i, n);
            dh[c].template load<TINY>(reinterpret_cast<const T*>(a.dh) + row * a.dhs, i, a.dh ? n : 0);
        }
        if (!whole)
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int i = (c * LANES + lane) * V;
                h[c].down(i, n);
                g[c].down(i, n);
                if (a.dh) dh[c].down(i, n);
            }
        float s = 0.f, sg = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const RowPiece<T> x(h[c]), y(g[c]), k(w[c]);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                s += x.x[e];
                sg = fmaf(y.x[e], k.x[e], sg);
            }
        }
        sums.over(s, sg);
        const float mu = s * rn;
        float q = 0.f, sx = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            h[c].again();
            g[c].again();
            w[c].again();
            const RowPiece<T> x(h[c]), y(g[c]), k(w[c]);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = (c * LANES + lane) * V + e < n ? x.x[e] - mu : 0.f;
                q = fmaf(d, d, q);
                sx = fmaf(d, y.x[e] * k.x[e], sx);
            }
        }
        sums.over(q, sx);
        const float inv = rsqrtf(q * rn + a.eps), mg = sg * rn, mx = sx * inv * rn;
        if (n == 0) continue;  // a row that is not there has an inv of its own: 0 times it need not be 0
#pragma unroll
        for (int c = 0; c < C; ++c) {
            h[c].again();
            g[c].again();
            w[c].again();
            const RowPiece<T> x(h[c]), y(g[c]), k(w[c]);
            RowPiece<T> d(dh[c]);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float xh = (x.x[e] - mu) * inv;
                dw[c][e] = fmaf(y.x[e], xh, dw[c][e]);  // (behind the row's end dy is 0)
                db[c][e] += y.x[e];
                d.x[e] += inv * (y.x[e] * k.x[e] - mg - xh * mx);
            }
            d.store(reinterpret_cast<T*>(a.dx) + row * a.n, (c * LANES + lane) * V, n);
        }
    }
    float* part = a.part + (size_t)blockIdx.x * 2 * a.n;
#pragma unroll
    for (int t = 0; t < 2; ++t, part += a.n) {
        if constexpr (ROWS == 1) {
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int i = (c * LANES + lane) * V + e;
                    if (i < a.n) part[i] = t ? db[c][e] : dw[c][e];
                }
        } else {
            if (t) __syncthreads();
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < V; ++e) folded[sub * WIDTH + (c * LANES + lane) * V + e] = t ? db[c][e] : dw[c][e];
            __syncthreads();
            for (int i = threadIdx.x; i < a.n; i += row_threads<LANES>()) {
                float s = 0.f;
#pragma unroll
                for (int k = 0; k < ROWS; ++k) s += folded[k * WIDTH + i];
                part[i] = s;
            }
        }
    }
}

// Rows of any length, a work-group each, read again for each step.
template <class T>
__global__ __launch_bounds__(1024) void layer_norm_forward_long_kernel(LayerNormCall a) {
    constexpr int V = RowPiece<T>::V;
    __shared__ float slots[2][2][16];
    RowSums<1024> sums{slots};
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = reinterpret_cast<const T*>(a.x) + row * a.xs;
        const T* r = a.res ? reinterpret_cast<const T*>(a.res) + row * a.rs : nullptr;
        T* h = a.res ? reinterpret_cast<T*>(a.h) + row * a.n : nullptr;
        float s = 0.f;
        RowPiece<T> p, o;
        for (long long i = threadIdx.x * V; i < a.n; i += 1024 * V) {
            p.load(x, (int)i, a.n);
            if (r) {
                o.load(r, (int)i, a.n);
#pragma unroll
                for (int e = 0; e < V; ++e) p.x[e] = (float)(T)(p.x[e] + o.x[e]);
                p.store(h, (int)i, a.n);
            }
#pragma unroll
            for (int e = 0; e < V; ++e) s += p.x[e];
        }
        const T* from = r ? h : x;  // of the stream each thread reads what it wrote
        const float mu = sums.over(s) / a.n;
        float q = 0.f;
        for (long long i = threadIdx.x * V; i < a.n; i += 1024 * V) {
            p.load(from, (int)i, a.n);
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (i + e < a.n) q = fmaf(p.x[e] - mu, p.x[e] - mu, q);
        }
        const float inv = rsqrtf(sums.over(q) / a.n + a.eps);
        for (long long i = threadIdx.x * V; i < a.n; i += 1024 * V) {
            RowPiece<T> w, b;
            p.load(from, (int)i, a.n);
            w.load(reinterpret_cast<const T*>(a.w), (int)i, a.n);
            if (a.b) b.load(reinterpret_cast<const T*>(a.b), (int)i, a.n);
            else b.clear();
#pragma unroll
            for (int e = 0; e < V; ++e) p.x[e] = fmaf((p.x[e] - mu) * inv, w.x[e], b.x[e]);
            p.store(reinterpret_cast<T*>(a.y) + row * a.n, (int)i, a.n);
        }
    }
}
template <class T>
__global__ __launch_bounds__(1024) void layer_norm_backward_long_kernel(LayerNormCall a) {
    constexpr int V = RowPiece<T>::V;
    __shared__ float slots[2][2][16];
    RowSums<1024> sums{slots};
    float* part = a.part + (size_t)blockIdx.x * 2 * a.n;  // each thread's own columns
    bool first = true;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, first = false) {
        const T* x = reinterpret_cast<const T*>(a.x) + row * a.xs;
        const T* dy = reinterpret_cast<const T*>(a.dy) + row * a.dys;
        float s = 0.f, sg = 0.f;
        RowPiece<T> h, g, w, d;
        for (long long i = threadIdx.x * V; i < a.n; i += 1024 * V) {
            h.load(x, (int)i, a.n);
            g.load(dy, (int)i, a.n);
            w.load(reinterpret_cast<const T*>(a.w), (int)i, a.n);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                s += h.x[e];
                sg = fmaf(g.x[e], w.x[e], sg);
            }
        }
        sums.over(s, sg);
        const float mu = s / a.n;
        float q = 0.f, sx = 0.f;
        for (long long i = threadIdx.x * V; i < a.n; i += 1024 * V) {
            h.load(x, (int)i, a.n);
            g.load(dy, (int)i, a.n);
            w.load(reinterpret_cast<const T*>(a.w), (int)i, a.n);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if (i + e >= a.n) continue;
                q = fmaf(h.x[e] - mu, h.x[e] - mu, q);
                sx = fmaf(h.x[e] - mu, g.x[e] * w.x[e], sx);
            }
        }
        sums.over(q, sx);
        const float inv = rsqrtf(q / a.n + a.eps), mg = sg / a.n, mx = sx * inv / a.n;
        for (long long i = threadIdx.x * V; i < a.n; i += 1024 * V) {
            h.load(x, (int)i, a.n);
            g.load(dy, (int)i, a.n);
            w.load(reinterpret_cast<const T*>(a.w), (int)i, a.n);
            if (a.dh) d.load(reinterpret_cast<const T*>(a.dh) + row * a.dhs, (int)i, a.n);
            else d.clear();
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if (i + e >= a.n) continue;
                const float xh = (h.x[e] - mu) * inv;
                part[i + e] = fmaf(g.x[e], xh, first ? 0.f : part[i + e]);
                part[a.n + i + e] = g.x[e] + (first ? 0.f : part[a.n + i + e]);
                d.x[e] += inv * (g.x[e] * w.x[e] - mg - xh * mx);
            }
            d.store(reinterpret_cast<T*>(a.dx) + row * a.n, (int)i, a.n);
        }
    }
}

// dw and db, 16 columns (one line of 64 bytes) at a time, so that narrow rows still spread over CUs: 64 threads to a column take every
// 64th part, four loads in flight, and add up in a fixed order.  part: [groups][2][n], of which the first `columns` of 2 n are wanted.
template <class T>
__global__ __launch_bounds__(1024) void layer_norm_weight_kernel(const float* __restrict__ part, T* __restrict__ dw, T* __restrict__ db,
                                                                 int groups, int n, int columns) {
    __shared__ float s[64][17];
    const int l = threadIdx.x & 15, w = threadIdx.x >> 4;
    const size_t step = 2 * (size_t)n;
    for (int first = blockIdx.x * 16; first < columns; first += gridDim.x * 16) {
        float v = 0.f;
        if (first + l < columns) {
            const float* p = part + first + l;
            int g = w;
            for (; g + 192 < groups; g += 256) {
                const float x0 = p[g * step], x1 = p[(g + 64) * step], x2 = p[(g + 128) * step], x3 = p[(g + 192) * step];
                v += (x0 + x1) + (x2 + x3);
            }
            for (; g < groups; g += 64) v += p[g * step];
        }
        s[w][l] = v;
        __syncthreads();
        if (w < 16) {  // thread (w, l): column w, parts l, l + 16, ...
            v = (s[l][w] + s[l + 16][w]) + (s[l + 32][w] + s[l + 48][w]);
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) v += __shfl_xor(v, o, 64);
            const int c = first + w;
            if (l == 0 && c < columns) (c < n ? dw : db)[c < n ? c : c - n] = (T)v;
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------------------------------------
typedef spion_layer_norm LayerNorm;

// Lanes to a row and pieces to a lane: the fewest lanes whose registers hold it.  (Three pieces beside two and four, bf16, a step: 16352 x 1026 85 us
// without, 74 with them; 14475 x 1159 70 and 60; 2653 x 5000 70 and 64.  bf16 rows past 16384 would spill in the backward, with
// six tensors' pieces of eight floats.)
struct RowShape {
    int lanes, pieces;  // 0: longer than the registers of a work-group
};
static RowShape row_shape(const LayerNorm& c, bool backward) {
    static const RowShape of[] = {{8, 1}, {16, 1}, {16, 2}, {64, 1}, {64, 2}, {64, 3}, {64, 4}, {256, 2}, {256, 3}, {256, 4}, {1024, 2}, {1024, 4}};
    for (const RowShape& s : of)
        if (c.width <= (long long)s.lanes * s.pieces * (c.bf16 ? 8 : 4) && !(backward && c.bf16 && s.lanes == 1024 && s.pieces == 4)) return s;
    return {0, 0};
}
static int rows_at_once(const RowShape& s) { return s.lanes == 0 || s.lanes >= 256 ? 1 : 256 / s.lanes; }
static long long row_groups(long long rows, int at_a_time, int per_cu) {
    return std::max(1LL, std::min((rows + at_a_time - 1) / at_a_time, (long long)per_cu * device_cus()));
}
// Work-groups of a backward.  Each leaves partial sums of 2 n floats, so beyond one for each CU no more than one for eight rows.  Three to a CU, four
// where a row has few lanes (a step with 2 / 3 / 4, us: 8192 x 4096 bf16 118 / 118 / 124, 16384 x 1000 58 / 55 / 60, 262144 x 64 90 / 76 / 69).
static long long layer_norm_groups(const LayerNorm& c) {
    const RowShape s = row_shape(c, true);
    return std::min(row_groups(c.rows, rows_at_once(s), s.lanes > 0 && s.lanes < 64 ? 4 : 3), std::max<long long>(device_cus(), c.rows / 8));
}

template <class T, int LANES, int C, bool TINY = false>
static bool run_rows(const LayerNormCall& a, bool backward, long long groups, hipStream_t stream) {
    const dim3 grid((unsigned)groups), block(row_threads<LANES>());
    if (!backward) {
        hipLaunchKernelGGL((layer_norm_forward_kernel<T, LANES, C, TINY>), grid, block, 0, stream, a);
        return check_launch("layer_norm_forward_kernel");
    }
    if constexpr (sizeof(T) == 4 || LANES * C < 4096) hipLaunchKernelGGL((layer_norm_backward_kernel<T, LANES, C, TINY>), grid, block, 0, stream, a);
    return check_launch("layer_norm_backward_kernel");
}
template <class T>
static bool run_layer_norm(const LayerNorm& c, bool backward, hipStream_t stream) {
    LayerNormCall a{};
    a.x = c.x, a.res = c.residual, a.w = c.weight, a.b = c.bias, a.dy = c.dy, a.dh = c.dh;
    a.y = c.y, a.h = c.h, a.dx = c.dx, a.part = c.workspace;
    a.rows = c.rows, a.xs = c.x_stride, a.rs = c.residual_stride, a.dys = c.dy_stride, a.dhs = c.dh_stride;
    a.n = c.width, a.eps = c.eps;
    const RowShape s = row_shape(c, backward);
    const long long groups = backward ? layer_norm_groups(c) : row_groups(c.rows, rows_at_once(s), s.lanes == 0 || s.lanes >= 256 ? 8 : 16);
    bool ok = false;
    switch (s.lanes * 8 + s.pieces) {
        case 8 * 8 + 1:
            ok = c.width < RowPiece<T>::V ? run_rows<T, 8, 1, true>(a, backward, groups, stream) : run_rows<T, 8, 1>(a, backward, groups, stream);
            break;
        case 16 * 8 + 1: ok = run_rows<T, 16, 1>(a, backward, groups, stream); break;
        case 16 * 8 + 2: ok = run_rows<T, 16, 2>(a, backward, groups, stream); break;
        case 64 * 8 + 1: ok = run_rows<T, 64, 1>(a, backward, groups, stream); break;
        case 64 * 8 + 2: ok = run_rows<T, 64, 2>(a, backward, groups, stream); break;
        case 64 * 8 + 3: ok = run_rows<T, 64, 3>(a, backward, groups, stream); break;
        case 64 * 8 + 4: ok = run_rows<T, 64, 4>(a, backward, groups, stream); break;
        case 256 * 8 + 2: ok = run_rows<T, 256, 2>(a, backward, groups, stream); break;
        case 256 * 8 + 3: ok = run_rows<T, 256, 3>(a, backward, groups, stream); break;
        case 256 * 8 + 4: ok = run_rows<T, 256, 4>(a, backward, groups, stream); break;
        case 1024 * 8 + 2: ok = run_rows<T, 1024, 2>(a, backward, groups, stream); break;
        case 1024 * 8 + 4: ok = run_rows<T, 1024, 4>(a, backward, groups, stream); break;
        default:
            if (backward) hipLaunchKernelGGL((layer_norm_backward_long_kernel<T>), dim3((unsigned)groups), dim3(1024), 0, stream, a);
            else hipLaunchKernelGGL((layer_norm_forward_long_kernel<T>), dim3((unsigned)groups), dim3(1024), 0, stream, a);
            ok = check_launch(backward ? "layer_norm_backward_long_kernel" : "layer_norm_forward_long_kernel");
    }
    if (!ok || !backward) return ok;
    const int columns = c.dbias ? 2 * c.width : c.width;
    hipLaunchKernelGGL((layer_norm_weight_kernel<T>), dim3((unsigned)std::min((columns + 15) / 16, 1 << 18)), dim3(1024), 0, stream, c.workspace,
                       reinterpret_cast<T*>(c.dweight), reinterpret_cast<T*>(c.dbias), (int)groups, c.width, columns);
    return check_launch("layer_norm_weight_kernel");
}

static bool layer_norm_sizes(const char* who, const LayerNorm* c) {
    if (!c) {
        set_error("%s: null pointer", who);
        return false;
    }
    if (c->rows < 1 || c->width < 1 || c->rows > (1LL << 40) || c->width > (1 << 29)) {
        set_error("%s: positive sizes expected, rows up to 2^40, a width up to 2^29", who);
        return false;
    }
    if (c->x_stride < 0 || c->residual_stride < 0 || c->dy_stride < 0 || c->dh_stride < 0 || !(c->eps >= 0.f)) {
        set_error("%s: strides and eps are not negative", who);
        return false;
    }
    return true;
}

long long layer_norm_workspace(const LayerNorm* c) {
    if (!layer_norm_sizes("spion_layer_norm_workspace", c)) return -1;
    return layer_norm_groups(*c) * 2 * c->width;
}
int layer_norm_forward(const LayerNorm* c, hipStream_t stream) {
    const char* who = "spion_layer_norm_forward";
    if (!layer_norm_sizes(who, c)) return 1;
    if (!c->x || !c->weight || !c->y || (c->residual && !c->h)) {
        set_error("%s: x, weight, y and, with a residual, the stream expected", who);
        return 1;
    }
    return (c->bf16 ? run_layer_norm<__bf16>(*c, false, stream) : run_layer_norm<float>(*c, false, stream)) ? 0 : 1;
}
int layer_norm_backward(const LayerNorm* c, hipStream_t stream) {
    const char* who = "spion_layer_norm_backward";
    if (!layer_norm_sizes(who, c)) return 1;
    if (!c->x || !c->weight || !c->dy || !c->dx || !c->dweight || !c->workspace) {
        set_error("%s: null pointer", who);
        return 1;
    }
    if (c->workspace_floats < layer_norm_groups(*c) * 2 * c->width) {
        set_error("%s: workspace of %lld floats, %lld expected", who, c->workspace_floats, layer_norm_groups(*c) * 2 * c->width);
        return 1;
    }
    return (c->bf16 ? run_layer_norm<__bf16>(*c, true, stream) : run_layer_norm<float>(*c, true, stream)) ? 0 : 1;
}

}  // namespace spion

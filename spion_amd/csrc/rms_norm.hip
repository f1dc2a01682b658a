// Root-mean-square norm of rows with the residual's addition ahead of it (the pre-norm encoder's other pass over the stream; the
// reference's layer has nn.LayerNorm there, models/model_transformer.py:55-102), its 8-bit form and its backward:
//   h = x + residual, rounded to the tensors' type: the stream as it goes on;   inv = 1 / sqrt(mean(h^2) + eps);   y = h inv w
//   8 bits: scale = max|y| / 448 of the unrounded row, codes = e4m3(y / scale), where 1 / rms cancels
//   dh = inv (dy w - h inv mean(dy w h inv)) + (gradient of the stream);   dw = sum over the rows of dy h inv
// Bound by memory: every tensor is read or written once where rows start on 16 bytes.  A row lies in the registers of 16, 64, 256 or
// 1024 lanes in pieces of 16 bytes (up to 16384 fp32 or 32768 bf16 elements), so the statistics need no second pass over it.  Where a
// width or stride is no multiple of 16 bytes a piece is one element, which holds rows of up to 4096; longer rows are read again
// for each step (from L2).  Statistics and sums are fp32.  Work-groups walk several rows each: the weight is read once, and the
// backward leaves one partial dw a work-group, which a second launch adds up in a fixed order.
// 262144 x 64 fp32: forward 45 us, backward 42 + 4; 8192 x 4096 bf16: 45 and 51 + 6; 16384 x 1000 bf16 to 8 bits: 20.  As many bytes at the
// 5062 GB/s of a copy of 1 GB: 53, 53 and 53, 53 and 23.  Off 16 bytes, bf16, calls: 16384 x 1001 25 us forward and 74 a step (1000: 21 and
// 73), 262144 x 65 39 and 114 (64: 23 and 74), 8192 x 4100 94 and 289 (4096: 41 and 105), 8192 x 5415 165 and 383 (5416: 73 and 170); fp32
// 262144 x 65 60 and 148 (64: 40 and 90), 8192 x 5415 201 and 452 (5416: 135 and 284).  The backward of bf16 rows past 16384 spills
// (424 bytes a lane): 1024 x 32768 312 us a step (2048 x 16384: 115).
#include "common.h"
#include "tile_ops.h"
#include "../../include/spion_hip.h"

#include <algorithm>
#include <climits>

namespace spion {

struct NormCall {
    const void *x, *res, *w, *dy, *dh;
    void *y, *h, *dx;
    unsigned char* codes;
    float *scales, *part;
    long long rows, xs, rs, dys, dhs;  // strides of rows, in elements; outputs are contiguous
    int n;
    float eps;
};

// V elements from memory as floats, and back
template <class T, int V>
struct Piece {
    float x[V];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (V == 1) {
            x[0] = (float)*p;
        } else {
            const u32x4 u = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 4) {
                    const unsigned bits = u[i];  // (a bit cast of a vector's element takes its first one)
                    x[i] = __builtin_bit_cast(float, bits);
                } else {
                    x[2 * i] = bf16_lo(u[i]);
                    x[2 * i + 1] = bf16_hi(u[i]);
                }
            }
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (V == 1) {
            *p = (T)x[0];
        } else {
            u32x4 u;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 4) u[i] = __builtin_bit_cast(unsigned, x[i]);
                else u[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
            }
            *reinterpret_cast<u32x4*>(p) = u;
        }
    }
    template <class Codes>
    __device__ __forceinline__ void store_codes(unsigned char* p, const Codes& of) const {
        if constexpr (V == 1) {
            *p = (unsigned char)__builtin_amdgcn_cvt_pk_fp8_f32(of(x[0]), 0.f, 0, false);
        } else {
            unsigned u[V / 4];
#pragma unroll
            for (int i = 0; i < V / 4; ++i) {
                int c = __builtin_amdgcn_cvt_pk_fp8_f32(of(x[4 * i]), of(x[4 * i + 1]), 0, false);
                u[i] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(of(x[4 * i + 2]), of(x[4 * i + 3]), c, true);
            }
            if constexpr (V == 4) *reinterpret_cast<unsigned*>(p) = u[0];
            else *reinterpret_cast<unsigned long long*>(p) = u[0] | (unsigned long long)u[V / 4 - 1] << 32;
        }
    }
};

// Sum (or maximum of bit patterns) over the LANES lanes of a row.  More than a wavefront: through LDS, two sets of slots taken in
// turn so that one barrier a reduction is enough.
template <int LANES>
struct RowReduce {
    float* slots;  // [2][16]
    int turn = 0;
    template <class F, class X>
    __device__ __forceinline__ X over(X v, F f) {
#pragma unroll
        for (int o = 1; o < (LANES < 64 ? LANES : 64); o <<= 1) v = f(v, __builtin_bit_cast(X, __shfl_xor(__builtin_bit_cast(int, v), o, 64)));
        if constexpr (LANES > 64) {
            X* s = reinterpret_cast<X*>(slots) + 16 * turn;
            turn ^= 1;
            if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
            __syncthreads();
            v = s[0];
#pragma unroll
            for (int i = 1; i < LANES / 64; ++i) v = f(v, s[i]);
        }
        return v;
    }
    __device__ __forceinline__ float sum(float v) {
        return over(v, [](float a, float b) { return a + b; });
    }
    __device__ __forceinline__ unsigned max_bits(unsigned v) {
        return over(v, [](unsigned a, unsigned b) { return a > b ? a : b; });
    }
};

constexpr float NORM_LEAST_SCALE = 0x1p-126f;
// 1 / rms as a power of two and what is left of it, in [1, 2).  The 8-bit form takes t = h 2^e w for the elements, which is exact for bf16
// (16 bits), and the rest for the scale alone: it cancels in the codes.
struct PowerAndRest {
    float power, rest;
    __device__ __forceinline__ explicit PowerAndRest(float inv) {
        power = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, inv) & 0x7f800000u);
        rest = power == 0.f ? 1.f : inv / power;  // (0: the squares' sum is infinite)
    }
};
// A row's scale and codes from max|t| by its bits, which order magnitudes and put NaN above infinity.  448 is e4m3's largest:
//   scale = max|t| rest / 448,   code = e4m3(448 t / max|t|) = e4m3((7/8 t) / (max|t| / 512))
// the quotient corrected by what it leaves, so that it is rounded once and ties of bf16 rows are ties (a rounded y over a rounded scale has
// 16 to 1000 codes of 2048 rows on their other side).  A row of zeros and rows whose scale would be below the least normal number have
// that for a scale, and their codes are exact or as fine as e4m3 is there.  An infinite max|t| has a reciprocal of 0 and nothing to
// correct.
struct RowCodes {
    float scale, num, den, by;
    bool correct;
    __device__ __forceinline__ RowCodes(unsigned bits, float rest) {
        const float most = __builtin_bit_cast(float, bits), s = most * rest / 448.f;
        const bool least = s < NORM_LEAST_SCALE;
        scale = least ? NORM_LEAST_SCALE : s;
        num = least ? rest : 0.875f;
        den = most * 0x1p-9f;
        by = least ? 0x1p126f : 1.f / den;
        correct = !least && by != 0.f;
    }
    __device__ __forceinline__ float operator()(float t) const {
        const float n = t * num, q = n * by;
        return correct ? fmaf(fmaf(-q, den, n), by, q) : q;
    }
};

// LANES lanes to a row of up to LANES * C * V elements; LANES <= 256: work-groups of 256 threads with 256 / LANES rows at a time.
template <int LANES>
constexpr int norm_threads() { return LANES < 256 ? 256 : LANES; }

template <class T, int V, int LANES, int C, bool F8>
__global__ __launch_bounds__(norm_threads<LANES>()) void norm_forward_kernel(NormCall a) {
    __shared__ float slots[32];
    constexpr int ROWS = norm_threads<LANES>() / LANES;
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    RowReduce<LANES> red{slots};
    Piece<T, V> w[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = (c * LANES + lane) * V;
        if (i < a.n) w[c].load(reinterpret_cast<const T*>(a.w) + i);
        else
#pragma unroll
            for (int e = 0; e < V; ++e) w[c].x[e] = 0.f;
    }
    const float rn = 1.f / a.n;
    for (long long r0 = (long long)blockIdx.x * ROWS; r0 < a.rows; r0 += (long long)gridDim.x * ROWS) {
        const long long row = r0 + sub;
        const bool there = row < a.rows;
        Piece<T, V> h[C];
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = (c * LANES + lane) * V;
            if (there && i < a.n) {
                h[c].load(reinterpret_cast<const T*>(a.x) + row * a.xs + i);
                if (a.res) {
                    Piece<T, V> r;
                    r.load(reinterpret_cast<const T*>(a.res) + row * a.rs + i);
#pragma unroll
                    for (int e = 0; e < V; ++e) h[c].x[e] = (float)(T)(h[c].x[e] + r.x[e]);
                    h[c].store(reinterpret_cast<T*>(a.h) + row * a.n + i);
                }
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) h[c].x[e] = 0.f;
            }
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) s = fmaf(h[c].x[e], h[c].x[e], s);
        const float inv = rsqrtf(red.sum(s) * rn + a.eps);
        const PowerAndRest parts(inv);
        const float by = F8 ? parts.power : inv;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) h[c].x[e] *= by * w[c].x[e];
        if constexpr (F8) {
            unsigned m = 0;
#pragma unroll
            for (int c = 0; c < C; ++c)
                if ((c * LANES + lane) * V < a.n)  // lanes without elements have 0 * inv, which may be NaN
#pragma unroll
                    for (int e = 0; e < V; ++e) m = max(m, __builtin_bit_cast(unsigned, h[c].x[e]) & 0x7fffffffu);
            const RowCodes codes(red.max_bits(m), parts.rest);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int i = (c * LANES + lane) * V;
                if (there && i < a.n) h[c].store_codes(a.codes + row * a.n + i, codes);
            }
            if (there && lane == 0) a.scales[row] = codes.scale;
        } else {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int i = (c * LANES + lane) * V;
                if (there && i < a.n) h[c].store(reinterpret_cast<T*>(a.y) + row * a.n + i);
            }
        }
    }
}

// a.x is the stream h.  part: [work-groups][n].
template <class T, int V, int LANES, int C>
__global__ __launch_bounds__(norm_threads<LANES>()) void norm_backward_kernel(NormCall a) {
    __shared__ float slots[32];
    constexpr int ROWS = norm_threads<LANES>() / LANES;
    __shared__ float sums[ROWS > 1 ? LANES * C * V * ROWS : 1];
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    RowReduce<LANES> red{slots};
    Piece<T, V> w[C];
    float dw[C][V];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = (c * LANES + lane) * V;
        if (i < a.n) w[c].load(reinterpret_cast<const T*>(a.w) + i);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (i >= a.n) w[c].x[e] = 0.f;
            dw[c][e] = 0.f;
        }
    }
    const float rn = 1.f / a.n;
    for (long long r0 = (long long)blockIdx.x * ROWS; r0 < a.rows; r0 += (long long)gridDim.x * ROWS) {
        const long long row = r0 + sub;
        const bool there = row < a.rows;
        Piece<T, V> h[C], g[C], d[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = (c * LANES + lane) * V;
            const bool in = there && i < a.n;
            if (in) {
                h[c].load(reinterpret_cast<const T*>(a.x) + row * a.xs + i);
                g[c].load(reinterpret_cast<const T*>(a.dy) + row * a.dys + i);
                if (a.dh) d[c].load(reinterpret_cast<const T*>(a.dh) + row * a.dhs + i);
            }
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if (!in) h[c].x[e] = g[c].x[e] = 0.f;
                if (!in || !a.dh) d[c].x[e] = 0.f;
            }
        }
        float ss = 0.f, sg = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                ss = fmaf(h[c].x[e], h[c].x[e], ss);
                sg = fmaf(h[c].x[e], g[c].x[e] * w[c].x[e], sg);
            }
        const float inv = rsqrtf(red.sum(ss) * rn + a.eps), m = red.sum(sg) * inv * rn;  // mean of dy w h inv
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = (c * LANES + lane) * V;
            if (!(there && i < a.n)) continue;  // a row that is not there has an inv of its own: 0 times it need not be 0
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float xh = h[c].x[e] * inv;
                dw[c][e] = fmaf(g[c].x[e], xh, dw[c][e]);
                d[c].x[e] += inv * (g[c].x[e] * w[c].x[e] - xh * m);
            }
            d[c].store(reinterpret_cast<T*>(a.dx) + row * a.n + i);
        }
    }
    float* part = a.part + (size_t)blockIdx.x * a.n;
    if constexpr (ROWS == 1) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int i = (c * LANES + lane) * V + e;
                if (i < a.n) part[i] = dw[c][e];
            }
    } else {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) sums[sub * LANES * C * V + (c * LANES + lane) * V + e] = dw[c][e];
        __syncthreads();
        for (int i = threadIdx.x; i < a.n; i += norm_threads<LANES>()) {
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < ROWS; ++k) s += sums[k * LANES * C * V + i];
            part[i] = s;
        }
    }
}

// Rows of any length, a work-group each, read again for each step.
template <class T, bool F8>
__global__ __launch_bounds__(1024) void norm_forward_long_kernel(NormCall a) {
    __shared__ float slots[32];
    RowReduce<1024> red{slots};
    const T* w = reinterpret_cast<const T*>(a.w);
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = reinterpret_cast<const T*>(a.x) + row * a.xs;
        const T* r = a.res ? reinterpret_cast<const T*>(a.res) + row * a.rs : nullptr;
        T* h = a.res ? reinterpret_cast<T*>(a.h) + row * a.n : nullptr;
        float s = 0.f;
        for (int i = threadIdx.x; i < a.n; i += 1024) {
            float v = (float)x[i];
            if (r) {
                const T sum = (T)(v + (float)r[i]);
                h[i] = sum;
                v = (float)sum;
            }
            s = fmaf(v, v, s);
        }
        const float inv = rsqrtf(red.sum(s) / a.n + a.eps);
        const PowerAndRest parts(inv);
        const float by = F8 ? parts.power : inv;
        auto y = [&](int i) {  // of this thread's own elements of h: they are its own writes
            return (float)(r ? h[i] : x[i]) * (by * (float)w[i]);
        };
        if constexpr (F8) {
            unsigned m = 0;
            for (int i = threadIdx.x; i < a.n; i += 1024) m = max(m, __builtin_bit_cast(unsigned, y(i)) & 0x7fffffffu);
            const RowCodes codes(red.max_bits(m), parts.rest);
            if (threadIdx.x == 0) a.scales[row] = codes.scale;
            for (int i = threadIdx.x; i < a.n; i += 1024) {
                Piece<T, 1> p;
                p.x[0] = y(i);
                p.store_codes(a.codes + row * a.n + i, codes);
            }
        } else {
            for (int i = threadIdx.x; i < a.n; i += 1024) {
                Piece<T, 1> p;
                p.x[0] = y(i);
                p.store(reinterpret_cast<T*>(a.y) + row * a.n + i);
            }
        }
    }
}
template <class T>
__global__ __launch_bounds__(1024) void norm_backward_long_kernel(NormCall a) {
    __shared__ float slots[32];
    RowReduce<1024> red{slots};
    const T* w = reinterpret_cast<const T*>(a.w);
    float* part = a.part + (size_t)blockIdx.x * a.n;
    for (int i = threadIdx.x; i < a.n; i += 1024) part[i] = 0.f;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* h = reinterpret_cast<const T*>(a.x) + row * a.xs;
        const T* g = reinterpret_cast<const T*>(a.dy) + row * a.dys;
        float ss = 0.f, sg = 0.f;
        for (int i = threadIdx.x; i < a.n; i += 1024) {
            const float v = (float)h[i];
            ss = fmaf(v, v, ss);
            sg = fmaf(v, (float)g[i] * (float)w[i], sg);
        }
        const float inv = rsqrtf(red.sum(ss) / a.n + a.eps), m = red.sum(sg) * inv / a.n;
        for (int i = threadIdx.x; i < a.n; i += 1024) {
            const float xh = (float)h[i] * inv, d = a.dh ? (float)reinterpret_cast<const T*>(a.dh)[row * a.dhs + i] : 0.f;
            part[i] = fmaf((float)g[i], xh, part[i]);
            reinterpret_cast<T*>(a.dx)[row * a.n + i] = (T)(d + inv * ((float)g[i] * (float)w[i] - xh * m));
        }
    }
}

// dw = sum of the work-groups' parts, 16 columns (one line of 64 bytes) at a time, so that narrow rows still spread over CUs: 64
// threads to a column take every 64th part, four loads in flight, and add up in a fixed order.  (2^18 work-groups at most: a launch holds fewer
// than 2^32 threads, and rows are up to 2^29 wide.)
template <class T>
__global__ __launch_bounds__(1024) void norm_weight_kernel(const float* __restrict__ part, T* __restrict__ dw, int groups, int n) {
    __shared__ float s[64][17];
    const int l = threadIdx.x & 15, w = threadIdx.x >> 4;
    for (int first = blockIdx.x * 16; first < n; first += gridDim.x * 16) {
        float v = 0.f;
        if (first + l < n) {
            const float* p = part + first + l;
            int g = w;
            for (; g + 192 < groups; g += 256) {
                const float x0 = p[(size_t)g * n], x1 = p[(size_t)(g + 64) * n], x2 = p[(size_t)(g + 128) * n], x3 = p[(size_t)(g + 192) * n];
                v += (x0 + x1) + (x2 + x3);
            }
            for (; g < groups; g += 64) v += p[(size_t)g * n];
        }
        s[w][l] = v;
        __syncthreads();
        if (w < 16) {  // thread (w, l): column w, parts l, l + 16, ...
            v = (s[l][w] + s[l + 16][w]) + (s[l + 32][w] + s[l + 48][w]);
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) v += __shfl_xor(v, o, 64);
            if (l == 0 && first + w < n) dw[first + w] = (T)v;
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------------------------------------
typedef spion_rms_norm Call;

// Lanes to a row and pieces to a lane: the fewest lanes whose registers hold it.
struct NormShape {
    int lanes, pieces;  // 0: longer than the registers of a work-group
};
static NormShape norm_shape(int n, int v) {
    static const NormShape of[] = {{16, 1}, {16, 2}, {64, 1}, {64, 2}, {64, 4}, {256, 2}, {256, 4}, {1024, 2}, {1024, 4}};
    for (const NormShape& s : of)
        if (n <= (long long)s.lanes * s.pieces * v) return s;
    return {0, 0};
}
// Elements of a piece: 16 bytes where every row of every tensor of the call starts on 16 bytes, else one.
static int norm_piece(const Call& c, bool backward) {
    const int v = c.bf16 ? 8 : 4;
    bool ok = c.width % v == 0 && c.x_stride % v == 0 && (c.residual == nullptr || c.residual_stride % v == 0);
    for (const void* p : {c.x, c.residual, c.weight}) ok = ok && reinterpret_cast<uintptr_t>(p) % 16 == 0;
    if (backward) {
        ok = ok && c.dy_stride % v == 0 && (c.dh == nullptr || c.dh_stride % v == 0);
        for (const void* p : {c.dy, c.dh, (const void*)c.dx}) ok = ok && reinterpret_cast<uintptr_t>(p) % 16 == 0;
    } else {
        for (const void* p : {(const void*)c.y, (const void*)c.h, (const void*)c.codes}) ok = ok && reinterpret_cast<uintptr_t>(p) % 16 == 0;
    }
    return ok ? v : 1;
}

static long long norm_groups(long long rows, int at_a_time, int per_cu) {
    return std::max(1LL, std::min((rows + at_a_time - 1) / at_a_time, (long long)per_cu * device_cus()));
}
// Work-groups of a backward.  Each leaves a partial dw of n floats, so beyond one for each CU no more than one for eight rows.
static long long backward_groups(long long rows, int n, int at_a_time) {
    const long long most = std::max<long long>(device_cus(), rows / 8);
    return std::min(norm_groups(rows, at_a_time, 4), most);
}
static int rows_at_a_time(const NormShape& s) { return s.lanes == 0 || s.lanes >= 256 ? 1 : 256 / s.lanes; }

template <class T, int V, int LANES, int C>
static bool run_shape(const Call& c, const NormCall& a, bool backward, long long groups, hipStream_t stream) {
    const dim3 grid((unsigned)groups), block(norm_threads<LANES>());
    if (backward) hipLaunchKernelGGL((norm_backward_kernel<T, V, LANES, C>), grid, block, 0, stream, a);
    else if (c.codes) hipLaunchKernelGGL((norm_forward_kernel<T, V, LANES, C, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((norm_forward_kernel<T, V, LANES, C, false>), grid, block, 0, stream, a);
    return check_launch(backward ? "norm_backward_kernel" : "norm_forward_kernel");
}
template <class T, int V>
static bool run_piece(const Call& c, const NormCall& a, bool backward, hipStream_t stream, long long& groups) {
    const NormShape s = norm_shape(c.width, V);
    const int rows = rows_at_a_time(s);
    groups = backward ? backward_groups(c.rows, c.width, rows) : norm_groups(c.rows, rows, s.lanes >= 256 ? 8 : 16);
    switch (s.lanes * 8 + s.pieces) {
        case 16 * 8 + 1: return run_shape<T, V, 16, 1>(c, a, backward, groups, stream);
        case 16 * 8 + 2: return run_shape<T, V, 16, 2>(c, a, backward, groups, stream);
        case 64 * 8 + 1: return run_shape<T, V, 64, 1>(c, a, backward, groups, stream);
        case 64 * 8 + 2: return run_shape<T, V, 64, 2>(c, a, backward, groups, stream);
        case 64 * 8 + 4: return run_shape<T, V, 64, 4>(c, a, backward, groups, stream);
        case 256 * 8 + 2: return run_shape<T, V, 256, 2>(c, a, backward, groups, stream);
        case 256 * 8 + 4: return run_shape<T, V, 256, 4>(c, a, backward, groups, stream);
        case 1024 * 8 + 2: return run_shape<T, V, 1024, 2>(c, a, backward, groups, stream);
        case 1024 * 8 + 4: return run_shape<T, V, 1024, 4>(c, a, backward, groups, stream);
        default: break;
    }
    const dim3 grid((unsigned)groups), block(1024);
    if (backward) hipLaunchKernelGGL((norm_backward_long_kernel<T>), grid, block, 0, stream, a);
    else if (c.codes) hipLaunchKernelGGL((norm_forward_long_kernel<T, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((norm_forward_long_kernel<T, false>), grid, block, 0, stream, a);
    return check_launch(backward ? "norm_backward_long_kernel" : "norm_forward_long_kernel");
}
template <class T>
static bool run_norm(const Call& c, bool backward, hipStream_t stream) {
    NormCall a{};
    a.x = c.x, a.res = c.residual, a.w = c.weight, a.dy = c.dy, a.dh = c.dh;
    a.y = c.y, a.h = c.h, a.dx = c.dx, a.codes = c.codes, a.scales = c.scales, a.part = c.workspace;
    a.rows = c.rows, a.xs = c.x_stride, a.rs = c.residual_stride, a.dys = c.dy_stride, a.dhs = c.dh_stride;
    a.n = c.width, a.eps = c.eps;
    long long groups = 0;
    const bool ok = norm_piece(c, backward) == 1 ? run_piece<T, 1>(c, a, backward, stream, groups)
                                                 : run_piece<T, 16 / sizeof(T)>(c, a, backward, stream, groups);
    if (!ok || !backward) return ok;
    hipLaunchKernelGGL((norm_weight_kernel<T>), dim3(std::min((c.width + 15) / 16, 1 << 18)), dim3(1024), 0, stream, c.workspace, reinterpret_cast<T*>(c.dweight),
                       (int)groups, c.width);
    return check_launch("norm_weight_kernel");
}

static bool norm_sizes(const char* who, const Call* c) {
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

// what any of the shapes a backward of these sizes may take needs: one that is not aligned takes the fewest rows at a time
long long norm_workspace(const Call* c) {
    if (!norm_sizes("spion_rms_norm_workspace", c)) return -1;
    return backward_groups(c->rows, c->width, 1) * c->width;
}
int norm_forward(const Call* c, hipStream_t stream) {
    const char* who = "spion_rms_norm_forward";
    if (!norm_sizes(who, c)) return 1;
    if (!c->x || !c->weight || (c->residual && !c->h) || (c->codes ? !c->scales || c->y : !c->y)) {
        set_error("%s: x, weight, the stream with a residual, and either y or codes with scales expected", who);
        return 1;
    }
    return (c->bf16 ? run_norm<__bf16>(*c, false, stream) : run_norm<float>(*c, false, stream)) ? 0 : 1;
}
int norm_backward(const Call* c, hipStream_t stream) {
    const char* who = "spion_rms_norm_backward";
    if (!norm_sizes(who, c)) return 1;
    if (!c->x || !c->weight || !c->dy || !c->dx || !c->dweight || !c->workspace) {
        set_error("%s: null pointer", who);
        return 1;
    }
    if (c->workspace_floats < backward_groups(c->rows, c->width, 1) * c->width) {
        set_error("%s: workspace of %lld floats, %lld expected", who, c->workspace_floats,
                  backward_groups(c->rows, c->width, 1) * c->width);
        return 1;
    }
    return (c->bf16 ? run_norm<__bf16>(*c, true, stream) : run_norm<float>(*c, true, stream)) ? 0 : 1;
}

}  // namespace spion

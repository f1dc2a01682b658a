// The kernels of bias_kernels.h for calls without a pattern that have queries (column pass: keys) enough to fill the machine with
// strips of 128 rows: each of a work-group's four wavefronts has 32 rows of its own, and the tiles of the other side are staged once
// for all four, in two buffers taken in turn (one barrier a stage).  That is a quarter of the reads from L2, and of the work-groups
// whose tables are set up and folded, and nothing is merged at the end.
#pragma once
#include "bias_kernels.h"

namespace spion {

// A stage: SUBS tiles of 32 rows of two tensors (K and V; Q and dO).  fp32 heads of 64 features have one tile a stage: their
// images take three times the LDS.
template <class T, int D>
struct BiasStage {
    typedef BiasTile<T, D> TL;
    static constexpr int SUBS = sizeof(T) == 4 && D == 64 ? 1 : 2, ROWS = 32 * SUBS;
    static constexpr int BYTES = 2 * SUBS * TL::BYTES;  // the first tensor's tiles, then the second's
    static constexpr int N = ROWS * TL::CPR / 256;      // pieces of each tensor a thread moves
    static_assert(N * 256 == ROWS * TL::CPR, "whole pieces");
    PieceInFlight<T> x[N], y[N];
    __device__ __forceinline__ void load(const char* xh, long long xld, const char* yh, long long yld, int first, int rows, int tid) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int n = 256 * i + tid, r = min(first + n / TL::CPR, rows - 1), c = n % TL::CPR;
            x[i].load(xh + r * xld + 8 * c * sizeof(T));
            y[i].load(yh + r * yld + 8 * c * sizeof(T));
        }
    }
    // word[s]: which rows of tile s take part
    __device__ __forceinline__ void store(char* buf, const unsigned (&word)[SUBS], int tid) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int n = 256 * i + tid, r = n / TL::CPR, c = n % TL::CPR, s = r >> 5;
            const bool there = ((SUBS == 2 && s ? word[SUBS - 1] : word[0]) >> (r & 31)) & 1u;
            x[i].template store<D>(buf + s * TL::BYTES, r & 31, c, there);
            y[i].template store<D>(buf + (SUBS + s) * TL::BYTES, r & 31, c, there);
        }
    }
};

template <class T, int D>
constexpr int bias_stages_bytes() {
    const int stages = 2 * BiasStage<T, D>::BYTES, merge = merge_floats<D>() * 4;
    return stages > merge ? stages : merge;
}

// The stages of the other side, one after the other: the list's with a key mask, all of them without.  body(stage's first row, words).
template <class T, int D, bool KEYS, class Store, class Body>
__device__ __forceinline__ void walk_stages(const BiasCall& a, ScanLds& sc, int b, int rows, const char* xh, long long xld,
                                            const char* yh, long long yld, char* lds, int tid, Store&& fetched, Body&& body) {
    typedef BiasStage<T, D> ST;
    const bool listed = KEYS && a.mask;
    const int tiles = (rows + 31) / 32, chunk = listed ? CHUNK : tiles;
    int parity = 0, none = 0;
    if (!listed) __syncthreads();  // the tables are there
    for (int first = 0; first < tiles; first += chunk) {
        const int count = min(chunk, tiles - first);
        const int n = listed ? scan_chunk<true, ST::SUBS>(a, sc, b, 0, first, count, tid, none) : (count + ST::SUBS - 1) / ST::SUBS;
        auto unit = [&](int i) __attribute__((always_inline)) { return (listed ? uniform(sc.list[i]) : i) * ST::SUBS; };
        ST st;
        int u = 0;
        if (n > 0) {
            u = unit(0);
            st.load(xh, xld, yh, yld, (first + u) * 32, rows, tid);
            fetched.load((first + u) * 32);
        }
        for (int i = 0; i < n; ++i, parity ^= 1) {
            unsigned word[ST::SUBS];
#pragma unroll
            for (int s = 0; s < ST::SUBS; ++s)
                word[s] = listed ? (u + s < count ? uniform(sc.words[u + s]) : 0u) : tail_word(rows - (first + u + s) * 32);
            char* buf = lds + parity * ST::BYTES;
            st.store(buf, word, tid);
            fetched.store(parity);
            __syncthreads();
            const int row0 = (first + u) * 32;
            if (i + 1 < n) {
                u = unit(i + 1);
                st.load(xh, xld, yh, yld, (first + u) * 32, rows, tid);
                fetched.load((first + u) * 32);
            }
            body(row0, word, buf, parity);
        }
    }
}
struct NothingElse {
    __device__ __forceinline__ void load(int) {}
    __device__ __forceinline__ void store(int) {}
};

// A wavefront's 32 x D result acc[c][r] (lane (li, h): row li, feature 32 c + acc_row(r, h)), scaled by the lane's f, through its part of
// red; out(row, eighth, values).
template <int D, class Out>
__device__ __forceinline__ void store_strip(const f32x16 (&acc)[D / 32], float f, float* red, int w, int l, Out&& out) {
    const int li = l & 31, h = l >> 5;
    float* mine = red + w * 32 * (D + 4);
    wave_lds_order();
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<f32x4*>(mine + li * (D + 4) + 32 * c + 8 * g + 4 * h) =
                f32x4{acc[c][4 * g] * f, acc[c][4 * g + 1] * f, acc[c][4 * g + 2] * f, acc[c][4 * g + 3] * f};
    wave_lds_order();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = 8 * i + (l >> 3), j = l & 7;
        float x[D / 8];
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(mine + row * (D + 4) + j * (D / 8) + 4 * k);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * k + e] = v[e];
        }
        out(row, j, x);
    }
}

template <class T, int D>
__global__ __launch_bounds__(256, 2) void bias_forward_dense_kernel(BiasCall a) {
    typedef BiasTile<T, D> TL;
    typedef BiasStage<T, D> ST;
    constexpr int SUBS = ST::SUBS;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float* tab = reinterpret_cast<float*>(lds + bias_stages_bytes<T, D>());
    ScanLds& sc = *reinterpret_cast<ScanLds*>(tab + bias_floats(a.R));
    const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, li = l & 31, h = l >> 5;
    const BiasItem it(a, gridDim.x);
    fill_bias<T>(a, it.h, tab, tid);
    const int q0 = it.strip * 128 + w * 32;
    const bool some = q0 < a.Lq;
    const typename TL::Row q = TL::load(a.q.head(it.b, it.h) + min(q0 + li, a.Lq - 1) * a.q.row, h, q0 + li < a.Lq);
    const typename TL::At at = TL::at(l);
    const float c2 = a.scale * LOG2E;
    const int qpos = q0 + a.off, far = 2 * (a.R + BIAS_PAD);

    f32x16 o[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) o[c] = splat16(0.f);
    float m = -__builtin_inff(), z = 0.f;
    walk_stages<T, D, true>(a, sc, it.b, a.Lk, a.k.head(it.b, it.h), a.k.row, a.v.head(it.b, it.h), a.v.row, lds, tid, NothingElse(),
        [&](int k0, const unsigned (&word)[SUBS], const char* buf, int) __attribute__((always_inline)) {
            if (!some) return;
            f32x16 s[SUBS];
#pragma unroll
            for (int u = 0; u < SUBS; ++u) s[u] = TL::feat(TL::rows(buf + u * TL::BYTES, at), q);
            const int rel0 = k0 - qpos;
            bool whole = true;
#pragma unroll
            for (int u = 0; u < SUBS; ++u) whole = whole && word[u] == ~0u;
            float t[SUBS][16], mul = 1.f, add = 0.f, mt = -__builtin_inff();
            if (whole && (rel0 - 31 >= a.R || rel0 + 32 * SUBS - 1 <= -a.R)) {
                // one number for the bias of all pairs: the products as they are, scaled where they enter the exponential
                mul = c2;
                add = tab[rel0 > 0 ? far : 0];
#pragma unroll
                for (int u = 0; u < SUBS; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        t[u][r] = s[u][r];
                        mt = fmaxf(mt, s[u][r]);
                    }
                mt = fmaf(mt, c2, add);
            } else {
#pragma unroll
                for (int u = 0; u < SUBS; ++u) {
                    logits_of<true>(s[u], c2, tab, a.R, rel0 + 32 * u, li, h, word[u], t[u]);
#pragma unroll
                    for (int r = 0; r < 16; ++r) mt = fmaxf(mt, t[u][r]);
                }
            }
            mt = half_swap_max(mt);
            if (__any(mt > m + BIAS_LAZY)) {
                const float up = fmaxf(m, mt);
                const float f = up == m ? 1.f : __builtin_amdgcn_exp2f(m - up);  // equal: also -infinity twice
                m = up;
                z *= f;
#pragma unroll
                for (int c = 0; c < D / 32; ++c)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[c][r] *= f;
            }
            add -= m == -__builtin_inff() ? 0.f : m;
#pragma unroll
            for (int u = 0; u < SUBS; ++u) {
                float p[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    p[r] = __builtin_amdgcn_exp2f(fmaf(t[u][r], mul, add));
                    z += p[r];
                }
                TL::add_t(buf + (SUBS + u) * TL::BYTES, at, p, o);
            }
        });
    z = half_swap_sum(z);
    __syncthreads();  // the stages are done with
    if (!some) return;
    if (h == 0 && q0 + li < a.Lq)
        a.lse[(size_t)it.bh * a.Lq + q0 + li] = z > 0.f ? m + __builtin_amdgcn_logf(z) : __builtin_inff();
    store_strip<D>(o, z > 0.f ? 1.f / z : 0.f, reinterpret_cast<float*>(lds), w, l, [&](int row, int j, float (&x)[D / 8]) {
        if (q0 + row < a.Lq) store_eighth<T, D>(a.o, it.b, it.h, q0 + row, j, x);
    });
}

template <class T, int D>
__global__ __launch_bounds__(256, 2) void bias_backward_row_dense_kernel(BiasCall a) {
    typedef BiasTile<T, D> TL;
    typedef BiasStage<T, D> ST;
    constexpr int SUBS = ST::SUBS;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float* tab = reinterpret_cast<float*>(lds + bias_stages_bytes<T, D>());
    ScanLds& sc = *reinterpret_cast<ScanLds*>(tab + bias_floats(a.R));
    const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, li = l & 31, h = l >> 5;
    const BiasItem it(a, gridDim.x);
    fill_bias<T>(a, it.h, tab, tid);
    const int q0 = it.strip * 128 + w * 32, qi = min(q0 + li, a.Lq - 1);
    const bool some = q0 < a.Lq, there = q0 + li < a.Lq;
    const typename TL::Row q = TL::load(a.q.head(it.b, it.h) + qi * a.q.row, h, there);
    const typename TL::Row go = TL::load(a.dout.head(it.b, it.h) + qi * a.dout.row, h, there);
    const size_t stat = (size_t)it.bh * a.Lq + qi;
    const float lse = there ? a.lse[stat] : __builtin_inff();
    const float delta = half_swap_sum(TL::dot(go, TL::load(a.o.head(it.b, it.h) + qi * a.o.row, h, there)));
    const typename TL::At at = TL::at(l);
    const float c2 = a.scale * LOG2E;
    const int qpos = q0 + a.off;
    const f32x16 minus = splat16(-delta);
    f32x16 dq[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) dq[c] = splat16(0.f);
    float sum = 0.f;
    walk_stages<T, D, true>(a, sc, it.b, a.Lk, a.k.head(it.b, it.h), a.k.row, a.v.head(it.b, it.h), a.v.row, lds, tid, NothingElse(),
        [&](int k0, const unsigned (&word)[SUBS], const char* buf, int) __attribute__((always_inline)) {
            if (!some) return;
#pragma unroll
            for (int u = 0; u < SUBS; ++u) {
                if (word[u] == 0) continue;
                const char *tk = buf + u * TL::BYTES, *tv = buf + (SUBS + u) * TL::BYTES;
                const f32x16 s = TL::feat(TL::rows(tk, at), q);
                const f32x16 dp = TL::feat(TL::rows(tv, at), go, minus);  // dP - D
                const int rel0 = k0 + 32 * u - qpos;
                float ds[16];
                if (word[u] == ~0u && (rel0 - 31 >= a.R || rel0 + 31 <= -a.R)) {
                    const float add = tab[rel0 > 0 ? 2 * (a.R + BIAS_PAD) : 0] - lse;
#pragma unroll
                    for (int r = 0; r < 16; ++r) ds[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c2, add)) * dp[r];
                } else {
                    float t[16];
                    logits_of<true>(s, c2, tab, a.R, rel0, li, h, word[u], t);
#pragma unroll
                    for (int r = 0; r < 16; ++r) ds[r] = __builtin_amdgcn_exp2f(t[r] - lse) * dp[r];
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) sum += ds[r];
                TL::add_t(tk, at, ds, dq);
            }
        });
    sum = half_swap_sum(sum);
    if (h == 0 && there) a.delta[stat] = delta + sum;
    __syncthreads();  // the stages are done with
    if (some)
        store_strip<D>(dq, a.scale, reinterpret_cast<float*>(lds), w, l, [&](int row, int j, float (&x)[D / 8]) {
            if (q0 + row < a.Lq) store_eighth<T, D>(a.dq, it.b, it.h, q0 + row, j, x);
        });
}

// The stage's queries' lse, -D and, for tiles far behind and far ahead, what the outermost buckets' bias leaves of lse.
struct QueryStats {
    const float *lse, *delta;
    float* lds;  // [2][4][64]
    float behind, ahead;
    int rows, tid;
    float e = 0.f, d = 0.f;
    __device__ __forceinline__ void load(int first) {
        if (tid < 64) {
            const bool there = first + tid < rows;
            e = there ? lse[first + tid] : __builtin_inff();
            d = there ? delta[first + tid] : 0.f;
        }
    }
    __device__ __forceinline__ void store(int parity) {
        if (tid < 64) {
            float* s = lds + 256 * parity + tid;
            s[0] = e;
            s[64] = -d;
            s[128] = behind - e;
            s[192] = ahead - e;
        }
    }
};

template <class T, int D>
__global__ __launch_bounds__(256, 2) void bias_backward_col_dense_kernel(BiasCall a) {
    typedef BiasTile<T, D> TL;
    typedef BiasStage<T, D> ST;
    constexpr int SUBS = ST::SUBS;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float* tab = reinterpret_cast<float*>(lds + bias_stages_bytes<T, D>());
    ScanLds& sc = *reinterpret_cast<ScanLds*>(tab + bias_floats(a.R));
    HistLds hl(sc, a.R);
    float* stats = reinterpret_cast<float*>(lds + bias_stages_bytes<T, D>() + bias_floats(a.R) * 4 + sizeof(ScanLds) + HistLds::bytes(a.R));
    const int tid = threadIdx.x, w = tid >> 6, l = tid & 63, li = l & 31, h = l >> 5;
    const BiasItem it(a, gridDim.x);
    fill_bias<T>(a, it.h, tab, tid, hl.bucket);
    hl.clear(a.R, tid);
    const int k0 = it.strip * 128 + w * 32, ki = min(k0 + li, a.Lk - 1);
    const bool key = key_there(a, it.b, k0 + li), some = __any(key);  // false behind the last key
    const typename TL::Row k = TL::load(a.k.head(it.b, it.h) + ki * a.k.row, h, k0 + li < a.Lk);
    const typename TL::Row v = TL::load(a.v.head(it.b, it.h) + ki * a.v.row, h, k0 + li < a.Lk);
    DifferenceSums sums(hl, w, a.R, key);
    const typename TL::At at = TL::at(l);
    const float c2 = a.scale * LOG2E;
    f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) dk[c] = dv[c] = splat16(0.f);
    QueryStats qs{a.lse + (size_t)it.bh * a.Lq, a.delta + (size_t)it.bh * a.Lq, stats,
                  bias_weight<T>(a, bucket_at(a, -a.R), it.h), bias_weight<T>(a, bucket_at(a, a.R), it.h), a.Lq, tid};
    if (__syncthreads_or(some))
        walk_stages<T, D, false>(a, sc, it.b, a.Lq, a.q.head(it.b, it.h), a.q.row, a.dout.head(it.b, it.h), a.dout.row, lds, tid, qs,
            [&](int r0, const unsigned (&)[SUBS], const char* buf, int parity) __attribute__((always_inline)) {
                if (!some) return;
#pragma unroll
                for (int u = 0; u < SUBS; ++u) {
                    if (SUBS == 2 && r0 + 32 * u >= a.Lq) continue;
                    const char *tq = buf + u * TL::BYTES, *tg = buf + (SUBS + u) * TL::BYTES;
                    const float* st = stats + 256 * parity + 32 * u + 4 * h;
                    f32x16 dp;
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const f32x4 d = *reinterpret_cast<const f32x4*>(st + 64 + 8 * g);
#pragma unroll
                        for (int j = 0; j < 4; ++j) dp[4 * g + j] = d[j];
                    }
                    const f32x16 s = TL::feat(TL::rows(tq, at), k);
                    dp = TL::feat(TL::rows(tg, at), v, dp);  // dP - D
                    const int rel0 = k0 - r0 - 32 * u - a.off;  // of the tile's corner: lane li, row r has rel0 + li - r
                    const bool near = sums.touches(rel0);
                    float p[16], ds[16];
                    if (near) {
                        const float* bias = tab + rel0 + a.R + BIAS_PAD + li - 4 * h;
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const f32x4 e = *reinterpret_cast<const f32x4*>(st + 8 * g);
#pragma unroll
                            for (int j = 0; j < 4; ++j) p[4 * g + j] = fmaf(s[4 * g + j], c2, bias[-(8 * g + j)] - e[j]);
                        }
                    } else {
                        const float* x = st + (rel0 > 0 ? 192 : 128);
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const f32x4 e = *reinterpret_cast<const f32x4*>(x + 8 * g);
#pragma unroll
                            for (int j = 0; j < 4; ++j) p[4 * g + j] = fmaf(s[4 * g + j], c2, e[j]);
                        }
                    }
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        p[r] = __builtin_amdgcn_exp2f(p[r]);
                        ds[r] = p[r] * dp[r];
                    }
                    if (near) sums.near(rel0, ds, li, h);
                    else sums.far(rel0, ds);
                    TL::add_t(tg, at, p, dv);
                    TL::add_t(tq, at, ds, dk);
                }
            });
    sums.finish(l);
    __syncthreads();  // the stages are done with, the histograms whole
    float* red = reinterpret_cast<float*>(lds);
    const unsigned keys = (unsigned)__ballot(key);
    // (a key that is left out: what it holds has reached its own lane, and nothing else)
    store_strip<D>(dv, 1.f, red, w, l, [&](int row, int j, float (&x)[D / 8]) {
        if (k0 + row >= a.Lk) return;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) x[i] = key_bit(keys, row) ? x[i] : 0.f;
        store_eighth<T, D>(a.dv, it.b, it.h, k0 + row, j, x);
    });
    store_strip<D>(dk, a.scale, red, w, l, [&](int row, int j, float (&x)[D / 8]) {
        if (k0 + row >= a.Lk) return;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) x[i] = key_bit(keys, row) ? x[i] : 0.f;
        store_eighth<T, D>(a.dk, it.b, it.h, k0 + row, j, x);
    });
    fold_hists(hl.hist, hl.bucket, bias_entries(a.R), a.buckets, tid, a.part + ((size_t)it.bh * a.strips + it.strip) * a.buckets);
}

}  // namespace spion

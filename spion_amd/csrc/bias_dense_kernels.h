// The kernels of bias_kernels.h for calls with queries (column pass: keys) enough to fill the machine, without a pattern or with one
// whose blocks hold whole stages.  A work-group has 128 rows, 32 to each of its four wavefronts, and the tiles of the other side
// are staged once for all four, in two buffers taken in turn (one barrier a stage).  That is a quarter of the reads from L2 and
// of the splitting of fp32 values, and of the work-groups whose tables are set up and folded.  Where the strips alone do not
// fill the machine the other side of an fp32 call is cut into pieces; each leaves its sums in a slot of the workspace for every 32
// rows, and a second launch adds the pieces of a strip up in their order.  (Which calls: walk_of in relative_bias.hip.)
//
// What bounds them, 128 padded heads of 2048, bf16, d = 64: forward 169 us (610 TFLOP/s), row pass 226 (680), column pass 337 to 345 (600).
// The matrix units are busy for 31 to 33 % of it, the vector units for about half (exponentials, bias, conversions, sums), LDS has 0.3
// to 4 % conflicts, and memory moves 0.1 to 0.2 GB: two wavefronts a SIMD (three in the forward, for which it spills 20 bytes a
// lane) take turns, and what one waits for the others do not fill.  64 rows to a wavefront halve the LDS reads, and were slower
// for the registers they take (column pass 337 -> 449).  16 heads of 8192 with a tenth of their 64 x 64 blocks: 79, 106 and 145 us,
// of which 19, 30 and 45 are there without any block.  128 fp32 heads of 1024, d = 32: forward 121 to 127 us, matrix units 42 % busy.
// (Times of kernels by themselves, under the profiler; in a call they follow each other more closely: these steps take 657 to 699 us and
// 305, table included.)
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
    __device__ __forceinline__ void load(const HeadBuf& xh, const HeadBuf& yh, int first, int tid) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int n = 256 * i + tid, r = n / TL::CPR, c = n % TL::CPR;
            x[i].load(xh.r, xh.at(first, xh.at(r, 8 * c * (int)sizeof(T))));
            y[i].load(yh.r, yh.at(first, yh.at(r, 8 * c * (int)sizeof(T))));
        }
    }
    // word[s]: which rows of tile s take part
    __device__ __forceinline__ void store(char* buf, const unsigned (&word)[SUBS], int tid) const {
        if ((word[0] & word[SUBS - 1]) == ~0u) put<true>(buf, word, tid);
        else put<false>(buf, word, tid);
    }
    template <bool ALL>
    __device__ __forceinline__ void put(char* buf, const unsigned (&word)[SUBS], int tid) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int n = 256 * i + tid, r = n / TL::CPR, c = n % TL::CPR, s = r >> 5;
            const bool there = ((SUBS == 2 && s ? word[SUBS - 1] : word[0]) >> (r & 31)) & 1u;
            x[i].template store<D, ALL>(buf + s * TL::BYTES, r & 31, c, there);
            y[i].template store<D, ALL>(buf + (SUBS + s) * TL::BYTES, r & 31, c, there);
        }
    }
};

template <class T, int D>
constexpr int bias_stages_bytes() {
    const int stages = 2 * BiasStage<T, D>::BYTES, merge = merge_floats<D>() * 4;
    return stages > merge ? stages : merge;
}

// The rows of a work-group and which of them a wavefront has.  WIDE: 128, each wavefront 32 of its own and all tiles of a stage.  Else
// 64, which lie in one block of a pattern of 64 x 64 blocks: two wavefronts have the same 32 rows and each one tile of the
// stage's two, and their sums are added in LDS at the end.
template <bool WIDE>
struct StripRows {
    static constexpr int ROWS = WIDE ? 128 : 64;
    static __device__ __forceinline__ int first(int strip, int w) { return strip * ROWS + 32 * (WIDE ? w : w & 1); }
};
// acc of wavefronts w and w + 2, in the first; red: 64 x D floats.  A barrier for all wavefronts.
template <int D>
__device__ __forceinline__ void join_halves(f32x16 (&acc)[D / 32], float* red, int w, int l) {
    float* at = red + (w & 1) * 32 * D + 4 * l;
    if (w >= 2)
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<f32x4*>(at + 256 * (4 * c + g)) = f32x4{acc[c][4 * g], acc[c][4 * g + 1], acc[c][4 * g + 2], acc[c][4 * g + 3]};
    __syncthreads();
    if (w < 2)
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(at + 256 * (4 * c + g));
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[c][4 * g + j] += x[j];
            }
}

// The list of a chunk's stages, for a strip of 128 or 64 rows: those that have a key which takes part and lie in the pattern of one of the
// wavefronts' rows (a block holds whole stages, and a wavefront's 32 rows lie in one block).  in_pattern grows by the keys of
// the pattern of this wavefront's rows.
template <bool KEYS, int SUBS, bool WIDE>
__device__ __forceinline__ int scan_stages(const BiasCall& a, ScanLds& s, const BiasItem& it, int first, int count, int tid, int& in_pattern) {
    const int w = uniform(tid >> 6), l = tid & 63;
    __syncthreads();
    if (KEYS) scan_words(a, s, it.b, first, count, tid);
    constexpr int ROUNDS = CHUNK / SUBS / 256;
    bool act[ROUNDS];
    unsigned long long votes[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int i = tid + 256 * r, tile = first + i * SUBS;
        const bool in = i * SUBS < count;
        unsigned who = in ? 15u : 0u;
        if (in && a.mat) {
            const int t = tile * 32 / a.bs, last = (KEYS ? a.Lq : a.Lk) - 1;
            who = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int o = min(StripRows<WIDE>::first(it.strip, k), last) / a.bs;
                who |= a.mat[KEYS ? (size_t)o * a.nb + t : (size_t)t * a.nb + o] != 0.f ? 1u << k : 0u;
            }
        }
        act[r] = who != 0;
        if (KEYS && act[r]) {
            unsigned any = s.words[i * SUBS];
            if (SUBS == 2 && i * SUBS + 1 < count) any |= s.words[i * SUBS + 1];
            act[r] = any != 0;
        }
        votes[r] = __ballot(act[r]);
        if (in) s.who[i] = (unsigned char)who;
        if (KEYS && a.mat) {
            const int beyond = max(0, tile * 32 + 32 * SUBS - a.Lk);  // of the last stage
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const bool have = (who >> k) & 1u;
                const int cut = __any(have && beyond > 0) ? (32 * SUBS - 1 - (a.Lk - 1) % (32 * SUBS)) : 0;
                const int n = 32 * SUBS * __popcll(__ballot(have)) - cut;
                if (l == 0) s.pats[k][4 * r + w] = n;
            }
        }
        if (l == 0) s.seg[4 * r + w] = __popcll(votes[r]);
    }
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        int before = 0;
#pragma unroll
        for (int k = 0; k < 4 * ROUNDS; ++k) before += k < 4 * r + w ? s.seg[k] : 0;
        if (act[r]) s.list[before + __popcll(votes[r] & ((1ull << l) - 1))] = (unsigned short)(tid + 256 * r);
    }
#pragma unroll
    for (int k = 0; k < 4 * ROUNDS; ++k) {
        total += s.seg[k];
        if (KEYS && a.mat) in_pattern += s.pats[w][k];
    }
    __syncthreads();
    return total;
}

// The stages of a piece of the other side, one after the other: the list's with a key mask or a pattern, all of them without.
// body(stage's first row, words, buffer, its parity): for the wavefronts whose rows have the stage.
template <class T, int D, bool WIDE, bool KEYS, class Store, class Body>
__device__ __forceinline__ void walk_stages(const BiasCall& a, ScanLds& sc, const BiasItem& it, int rows, const HeadBuf& xh,
                                            const HeadBuf& yh, char* lds, int tid, int& in_pattern, Store&& fetched, Body&& body) {
    typedef BiasStage<T, D> ST;
    const bool listed = (KEYS && a.mask) || a.mat;
    const int w = uniform(tid >> 6);
    const int from = it.split * a.per_split, to = min((rows + 31) / 32, from + a.per_split), chunk = listed ? CHUNK : a.per_split;
    int parity = 0;
    if (!listed) __syncthreads();  // the tables are there
    for (int first = from; first < to; first += chunk) {
        const int count = min(chunk, to - first);
        const int n = listed ? scan_stages<KEYS, ST::SUBS, WIDE>(a, sc, it, first, count, tid, in_pattern) : (count + ST::SUBS - 1) / ST::SUBS;
        // Which stage comes after next, and its words, are read from LDS while a stage is worked on.
        struct Next {
            int unit;
            unsigned who, word[ST::SUBS];
        };
        auto look_up = [&](int i) __attribute__((always_inline)) {
            Next x;
            x.unit = listed ? (int)sc.list[min(i, n - 1)] : i;
            x.who = 15u;
            if (listed) {
                x.who = sc.who[x.unit];
#pragma unroll
                for (int s = 0; s < ST::SUBS; ++s) x.word[s] = KEYS ? sc.words[x.unit * ST::SUBS + s] : 0u;
            }
            return x;
        };
        ST st;
        Next next, after;
        if (n > 0) {
            next = look_up(0);
            next.unit = uniform(next.unit);
            st.load(xh, yh, (first + next.unit * ST::SUBS) * 32, tid);
            fetched.load((first + next.unit * ST::SUBS) * 32);
            after = look_up(1);
        }
        for (int i = 0; i < n; ++i, parity ^= 1) {
            const int u = next.unit * ST::SUBS, row0 = (first + u) * 32;
            unsigned word[ST::SUBS];
#pragma unroll
            for (int s = 0; s < ST::SUBS; ++s)
                word[s] = listed && KEYS ? (u + s < count ? (unsigned)uniform((int)next.word[s]) : 0u) : tail_word(rows - row0 - 32 * s);
            const bool mine = (uniform((int)next.who) >> w) & 1;
            char* buf = lds + parity * ST::BYTES;
            st.store(buf, word, tid);
            fetched.store(parity);
            __syncthreads();
            if (i + 1 < n) {
                next = after;
                next.unit = uniform(next.unit);
                st.load(xh, yh, (first + next.unit * ST::SUBS) * 32, tid);
                fetched.load((first + next.unit * ST::SUBS) * 32);
                after = look_up(i + 2);
            }
            if (mine) body(row0, word, buf, parity);
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

template <class T, int D, bool WIDE>
__global__ __launch_bounds__(256, (sizeof(T) == 2 ? 3 : 2)) void bias_forward_dense_kernel(BiasCall a) {
    typedef BiasTile<T, D> TL;
    typedef BiasStage<T, D> ST;
    constexpr int SUBS = ST::SUBS, MINE = WIDE ? SUBS : 1;  // tiles of a stage, and a wavefront's among them
    static_assert(WIDE || SUBS == 2, "a tile for each half");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float* tab = reinterpret_cast<float*>(lds + bias_stages_bytes<T, D>());
    ScanLds& sc = *reinterpret_cast<ScanLds*>(tab + bias_floats(a.R));
    const int tid = threadIdx.x, w = uniform(tid >> 6), l = tid & 63, li = l & 31, h = l >> 5;
    const BiasItem it(a, gridDim.x);
    fill_bias<T>(a, it.h, tab, tid);
    const int q0 = StripRows<WIDE>::first(it.strip, w), half = WIDE ? 0 : w >> 1;
    const bool some = q0 < a.Lq;
    const typename TL::Row q = TL::load(a.q.head(it.b, it.h) + min(q0 + li, a.Lq - 1) * a.q.row, h, q0 + li < a.Lq);
    const typename TL::At at = TL::at(l);
    const float c2 = a.scale * LOG2E;
    const int qpos = q0 + a.off, far = 2 * (a.R + BIAS_PAD);
    q.settled();

    f32x16 o[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) o[c] = splat16(0.f);
    float m = -__builtin_inff(), z = 0.f;
    int in_pattern = 0;
    walk_stages<T, D, WIDE, true>(a, sc, it, a.Lk, HeadBuf::of<T, D>(a.k, it.b, it.h, a.Lk), HeadBuf::of<T, D>(a.v, it.b, it.h, a.Lk), lds, tid, in_pattern, NothingElse(),
        [&](int k0, const unsigned (&words)[SUBS], const char* stage, int) __attribute__((always_inline)) {
            if (!some) return;
            const char* buf = stage + half * TL::BYTES;
            unsigned word[MINE];
#pragma unroll
            for (int u = 0; u < MINE; ++u) word[u] = WIDE ? words[u] : half ? words[SUBS - 1] : words[0];
            f32x16 s[MINE];
            typename TL::Row kr[MINE];
#pragma unroll
            for (int u = 0; u < MINE; ++u) kr[u] = TL::rows(buf + u * TL::BYTES, at);
            issue_order();
#pragma unroll
            for (int u = 0; u < MINE; ++u) s[u] = TL::feat(kr[u], q);
            const int rel0 = k0 + 32 * half - qpos;
            bool whole = true;
#pragma unroll
            for (int u = 0; u < MINE; ++u) whole = whole && word[u] == ~0u;
            float t[MINE][16], mul = 1.f, add = 0.f, mt = -__builtin_inff();
            if (whole && (rel0 - 31 >= a.R || rel0 + 32 * MINE - 1 <= -a.R)) {
                // one number for the bias of all pairs: the products as they are, scaled where they enter the exponential
                mul = c2;
                add = tab[rel0 > 0 ? far : 0];
#pragma unroll
                for (int u = 0; u < MINE; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        t[u][r] = s[u][r];
                        mt = fmaxf(mt, s[u][r]);
                    }
                mt = fmaf(mt, c2, add);
            } else {
#pragma unroll
                for (int u = 0; u < MINE; ++u) {
                    if (whole) logits_of<false>(s[u], c2, tab, a.R, rel0 + 32 * u, li, h, word[u], t[u]);
                    else logits_of<true>(s[u], c2, tab, a.R, rel0 + 32 * u, li, h, word[u], t[u]);
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
            for (int u = 0; u < MINE; ++u) {
                float p[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    p[r] = __builtin_amdgcn_exp2f(fmaf(t[u][r], mul, add));
                    z += p[r];
                }
                TL::add_t(TL::columns(buf + (SUBS + u) * TL::BYTES, at), p, o);
            }
        });
    z = half_swap_sum(z);
    if (!WIDE) {
        if (h == 0) sc.ml[w][0][li] = m, sc.ml[w][1][li] = z;
        __syncthreads();
        const float mo = sc.ml[w ^ 2][0][li], M = fmaxf(m, mo), base = M == -__builtin_inff() ? 0.f : M, f = __builtin_amdgcn_exp2f(m - base);
        z = z * f + sc.ml[w ^ 2][1][li] * __builtin_amdgcn_exp2f(mo - base);
        m = M;
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[c][r] *= f;
        join_halves<D>(o, reinterpret_cast<float*>(lds), w, l);
    }
    __syncthreads();  // the stages are done with
    if (!some || half) return;
    if (sizeof(T) == 4 && WIDE && a.splits > 1) {  // (bf16 strips and strips of 64 are never cut)
        float* slot = a.part + it.slot(a, w) * bias_slot<D>();
        if (h == 0) {
            slot[32 * D + li] = m;
            slot[32 * D + 32 + li] = z;
            slot[32 * D + 64 + li] = __builtin_bit_cast(float, in_pattern);
        }
        store_strip<D>(o, 1.f, reinterpret_cast<float*>(lds), w, l, [&](int row, int j, float (&x)[D / 8]) {
            store_values<float, D / 8>(reinterpret_cast<char*>(slot + row * D + j * (D / 8)), x);
        });
        return;
    }
    const int off = a.mat ? a.Lk - in_pattern : 0;  // keys off the pattern: a logit of 0 each
    float scale = 1.f;
    if (off > 0) {
        const float up = fmaxf(m, 0.f);
        scale = __builtin_amdgcn_exp2f(m - up);
        z = z * scale + off * __builtin_amdgcn_exp2f(-up);
        m = up;
    }
    if (h == 0 && q0 + li < a.Lq)
        a.lse[(size_t)it.bh * a.Lq + q0 + li] = z == 0.f ? __builtin_inff() : m + __builtin_amdgcn_logf(z);
    store_strip<D>(o, z == 0.f ? 0.f : scale / z, reinterpret_cast<float*>(lds), w, l, [&](int row, int j, float (&x)[D / 8]) {
        if (q0 + row < a.Lq) store_eighth<T, D>(a.o, it.b, it.h, q0 + row, j, x);
    });
}

// Sums of the same eight features (D = 64; four for 32) of `pieces` slots, in their order.
template <int D>
__device__ __forceinline__ void add_pieces(const float* p, int pieces, int stride, float (&x)[D / 8]) {
#pragma unroll
    for (int i = 0; i < D / 8; ++i) x[i] = 0.f;
#pragma unroll 4
    for (int k = 0; k < pieces; ++k)
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(p + (size_t)k * stride + 4 * i);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * i + e] += v[e];
        }
}

template <class T, int D, bool WIDE>
__global__ __launch_bounds__(256, (bias_waves<T, D>())) void bias_backward_row_dense_kernel(BiasCall a) {
    typedef BiasTile<T, D> TL;
    typedef BiasStage<T, D> ST;
    constexpr int SUBS = ST::SUBS, MINE = WIDE ? SUBS : 1;  // tiles of a stage, and a wavefront's among them
    static_assert(WIDE || SUBS == 2, "a tile for each half");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float* tab = reinterpret_cast<float*>(lds + bias_stages_bytes<T, D>());
    ScanLds& sc = *reinterpret_cast<ScanLds*>(tab + bias_floats(a.R));
    const int tid = threadIdx.x, w = uniform(tid >> 6), l = tid & 63, li = l & 31, h = l >> 5;
    const BiasItem it(a, gridDim.x);
    fill_bias<T>(a, it.h, tab, tid);
    const int q0 = StripRows<WIDE>::first(it.strip, w), half = WIDE ? 0 : w >> 1, qi = min(q0 + li, a.Lq - 1);
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
    q.settled();
    go.settled();
    f32x16 dq[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) dq[c] = splat16(0.f);
    float sum = 0.f;
    int in_pattern = 0;
    walk_stages<T, D, WIDE, true>(a, sc, it, a.Lk, HeadBuf::of<T, D>(a.k, it.b, it.h, a.Lk), HeadBuf::of<T, D>(a.v, it.b, it.h, a.Lk), lds, tid, in_pattern, NothingElse(),
        [&](int k0, const unsigned (&words)[SUBS], const char* buf, int) __attribute__((always_inline)) {
            if (!some) return;
#pragma unroll
            for (int n = 0; n < MINE; ++n) {
                const int u = WIDE ? n : half;
                const unsigned word = WIDE ? words[n] : half ? words[SUBS - 1] : words[0];
                if (word == 0) continue;
                const char *tk = buf + u * TL::BYTES, *tv = buf + (SUBS + u) * TL::BYTES;
                const typename TL::Row kr = TL::rows(tk, at), vr = TL::rows(tv, at);
                typename TL::Columns kt;
                issue_order();
                const f32x16 s = TL::feat(kr, q);
                const f32x16 dp = TL::feat(vr, go, minus);  // dP - D
                if (TL::EARLY) {
                    kt = TL::columns(tk, at);
                    read_behind_products<D / 8, D / 8>();
                }
                const int rel0 = k0 + 32 * u - qpos;
                float ds[16];
                if (word == ~0u && (rel0 - 31 >= a.R || rel0 + 31 <= -a.R)) {
                    const float add = tab[rel0 > 0 ? 2 * (a.R + BIAS_PAD) : 0] - lse;
#pragma unroll
                    for (int r = 0; r < 16; ++r) ds[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c2, add)) * dp[r];
                } else {
                    float t[16];
                    if (word == ~0u) logits_of<false>(s, c2, tab, a.R, rel0, li, h, word, t);
                    else logits_of<true>(s, c2, tab, a.R, rel0, li, h, word, t);
#pragma unroll
                    for (int r = 0; r < 16; ++r) ds[r] = __builtin_amdgcn_exp2f(t[r] - lse) * dp[r];
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) sum += ds[r];
                if (!TL::EARLY) kt = TL::columns(tk, at);
                TL::add_t(kt, ds, dq);
            }
        });
    sum = half_swap_sum(sum);
    __syncthreads();  // the stages are done with
    if (!WIDE) {
        if (h == 0) sc.ml[w][0][li] = sum;
        join_halves<D>(dq, reinterpret_cast<float*>(lds), w, l);
        sum += sc.ml[w ^ 2][0][li];
        __syncthreads();
    }
    if (!some || half) return;
    if (sizeof(T) == 4 && WIDE && a.splits > 1) {
        float* slot = a.part + it.slot(a, w) * bias_slot<D>();
        if (h == 0) {
            slot[32 * D + li] = sum;
            slot[32 * D + 32 + li] = delta;
            slot[32 * D + 64 + li] = __builtin_bit_cast(float, in_pattern);
        }
        store_strip<D>(dq, a.scale, reinterpret_cast<float*>(lds), w, l, [&](int row, int j, float (&x)[D / 8]) {
            store_values<float, D / 8>(reinterpret_cast<char*>(slot + row * D + j * (D / 8)), x);
        });
    } else {
        if (h == 0 && there) a.delta[stat] = exact_d<T>(delta, sum, lse, a.mat ? a.Lk - in_pattern : 0);
        store_strip<D>(dq, a.scale, reinterpret_cast<float*>(lds), w, l, [&](int row, int j, float (&x)[D / 8]) {
            if (q0 + row < a.Lq) store_eighth<T, D>(a.dq, it.b, it.h, q0 + row, j, x);
        });
    }
}

// The pieces of 32 rows of dQ and D.
template <class T, int D>
__global__ __launch_bounds__(256) void bias_merge_row_kernel(BiasCall a) {
    const int tid = threadIdx.x, row = tid >> 3, j = tid & 7;
    const int strips = (a.Lq + 31) / 32, strip = blockIdx.x % strips, bh = blockIdx.x / strips, q = strip * 32 + row;
    if (q >= a.Lq) return;
    const float* slot = a.part + (size_t)blockIdx.x * a.splits * bias_slot<D>();
    float x[D / 8];
    add_pieces<D>(slot + row * D + j * (D / 8), a.splits, bias_slot<D>(), x);
    store_eighth<T, D>(a.dq, bh / a.H, bh % a.H, q, j, x);
    if (j == 0) {
        float s = 0.f;
        int in_pattern = 0;
        for (int k = 0; k < a.splits; ++k) {
            s += slot[k * bias_slot<D>() + 32 * D + row];
            in_pattern += __builtin_bit_cast(int, slot[k * bias_slot<D>() + 32 * D + 64 + row]);
        }
        const size_t stat = (size_t)bh * a.Lq + q;
        a.delta[stat] = exact_d<T>(slot[32 * D + 32 + row], s, a.lse[stat], a.mat ? a.Lk - in_pattern : 0);
    }
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

template <class T, int D, bool WIDE>
__global__ __launch_bounds__(256, (bias_waves<T, D>())) void bias_backward_col_dense_kernel(BiasCall a) {
    typedef BiasTile<T, D> TL;
    typedef BiasStage<T, D> ST;
    constexpr int SUBS = ST::SUBS, MINE = WIDE ? SUBS : 1;  // tiles of a stage, and a wavefront's among them
    static_assert(WIDE || SUBS == 2, "a tile for each half");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float* tab = reinterpret_cast<float*>(lds + bias_stages_bytes<T, D>());
    ScanLds& sc = *reinterpret_cast<ScanLds*>(tab + bias_floats(a.R));
    HistLds hl(sc, a.R);
    float* stats = reinterpret_cast<float*>(lds + bias_stages_bytes<T, D>() + bias_floats(a.R) * 4 + sizeof(ScanLds) + HistLds::bytes(a.R));
    const int tid = threadIdx.x, w = uniform(tid >> 6), l = tid & 63, li = l & 31, h = l >> 5;
    const BiasItem it(a, gridDim.x);
    fill_bias<T>(a, it.h, tab, tid, hl.bucket);
    hl.clear(a.R, tid);
    const int k0 = StripRows<WIDE>::first(it.strip, w), half = WIDE ? 0 : w >> 1, ki = min(k0 + li, a.Lk - 1);
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
    k.settled();
    v.settled();
    int none = 0;
    if (__syncthreads_or(some))
        walk_stages<T, D, WIDE, false>(a, sc, it, a.Lq, HeadBuf::of<T, D>(a.q, it.b, it.h, a.Lq), HeadBuf::of<T, D>(a.dout, it.b, it.h, a.Lq), lds, tid, none, qs,
            [&](int r0, const unsigned (&)[SUBS], const char* buf, int parity) __attribute__((always_inline)) {
                if (!some) return;
#pragma unroll
                for (int n = 0; n < MINE; ++n) {
                    const int u = WIDE ? n : half;
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
                    const typename TL::Row qr = TL::rows(tq, at), gr = TL::rows(tg, at);
                    typename TL::Columns qt, gt;
                    issue_order();
                    const f32x16 s = TL::feat(qr, k);
                    dp = TL::feat(gr, v, dp);  // dP - D
                    if (TL::EARLY) {
                        gt = TL::columns(tg, at), qt = TL::columns(tq, at);
                        read_behind_products<D / 8, 2 * D / 8>();
                    }
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
                    if (!TL::EARLY) gt = TL::columns(tg, at);
                    TL::add_t(gt, p, dv);
                    if (!TL::EARLY) qt = TL::columns(tq, at);
                    TL::add_t(qt, ds, dk);
                    if (near) sums.near(rel0, ds, li, h);
                    else sums.far(rel0, ds);
                }
            });
    sums.finish(l);
    __syncthreads();  // the stages are done with, the histograms whole
    float* red = reinterpret_cast<float*>(lds);
    if (!WIDE) {
        join_halves<D>(dv, red, w, l);
        join_halves<D>(dk, red + 64 * D, w, l);
        __syncthreads();
    }
    const unsigned keys = (unsigned)__ballot(key);
    if (half) {  // (the other wavefront has both halves' sums)
    } else if (sizeof(T) == 4 && WIDE && a.splits > 1) {
        if (k0 < a.Lk) {
            float* slot = a.part + it.slot(a, w) * (2 * 32 * D);
            store_strip<D>(dv, 1.f, red, w, l, [&](int row, int j, float (&x)[D / 8]) {
                store_values<float, D / 8>(reinterpret_cast<char*>(slot + row * D + j * (D / 8)), x);
            });
            store_strip<D>(dk, a.scale, red, w, l, [&](int row, int j, float (&x)[D / 8]) {
                store_values<float, D / 8>(reinterpret_cast<char*>(slot + 32 * D + row * D + j * (D / 8)), x);
            });
        }
    } else {
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
    }
    fold_hists(hl.hist, hl.bucket, reinterpret_cast<int*>(hl.diag), bias_entries(a.R), a.buckets, tid,
               a.tables + (((size_t)it.bh * a.strips + it.strip) * a.splits + it.split) * a.buckets);
}

// The pieces of 32 rows of dV and dK.
template <class T, int D>
__global__ __launch_bounds__(256) void bias_merge_col_kernel(BiasCall a) {
    const int tid = threadIdx.x, row = tid >> 3, j = tid & 7;
    const int strips = (a.Lk + 31) / 32, strip = blockIdx.x % strips, bh = blockIdx.x / strips, b = bh / a.H, h = bh % a.H;
    const int key = strip * 32 + row;
    if (key >= a.Lk) return;
    const float* slot = a.part + (size_t)blockIdx.x * a.splits * (2 * 32 * D) + row * D + j * (D / 8);
    const bool keep = key_there(a, b, key);
    float x[D / 8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        add_pieces<D>(slot + t * 32 * D, a.splits, 2 * 32 * D, x);
#pragma unroll
        for (int i = 0; i < D / 8; ++i) x[i] = keep ? x[i] : 0.f;
        store_eighth<T, D>(t ? a.dk : a.dv, b, h, key, j, x);
    }
}

// -------------------------------------------------------------------------------------------------
// Mean probability map of all samples and heads
// -------------------------------------------------------------------------------------------------
// A work-group has 64 x 64 pairs of the map and goes through the samples of the heads, one head after the other; its wavefronts
// have a quarter of the pairs each.  Q and K of a pair of tiles are staged (and fp32 ones split) once for all four,
// probabilities are formed from the forward's lse, added up in registers and never written.  Where the tiles alone do not fill
// the machine the (head, sample) pairs are cut into pieces whose sums a second launch adds up.  (A tile of 32 x 32 a wavefront,
// operands straight from memory, bias and lse gathered for each pair: 275 us against 91, fp32, 128 heads of 1024.)
template <class T, int D>
constexpr int bias_mean_bytes() {
    const int tiles = 4 * BiasTile<T, D>::BYTES, map = 64 * 65 * 4;
    return tiles > map ? tiles : map;
}
template <class T, int D>
__global__ __launch_bounds__(256) void bias_mean_kernel(BiasCall a) {
    typedef BiasTile<T, D> TL;
    constexpr int N = 64 * TL::CPR / 256;  // pieces of each tensor a thread moves
    __shared__ __attribute__((aligned(16))) char lds[bias_mean_bytes<T, D>()];
    __shared__ float tab[128];  // the head's bias of differences -63 .. 63 from the tile's corner
    const int tid = threadIdx.x, w = uniform(tid >> 6), l = tid & 63, li = l & 31, h = l >> 5;
    const int kt = (a.Lk + 63) / 64, all = a.B * a.H;
    int tile = xcd_remap(blockIdx.x, gridDim.x);
    const int split = tile % a.splits;
    tile /= a.splits;
    const int q0 = tile / kt * 64, k0 = tile % kt * 64, qw = 32 * (w >> 1), kw = 32 * (w & 1);
    const int corner = k0 - q0 - a.off;
    const bool far = corner - 63 >= a.R || corner + 63 <= -a.R;  // one bucket
    const int bucket = bucket_at(a, corner + min(tid, 126) - 63);
    const float c2 = a.scale * LOG2E;
    const typename TL::At at = TL::at(l);
    const int q = q0 + qw + li;
    float sum[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) sum[r] = 0.f;

    PieceInFlight<T> x[N], y[N];
    float lse = 0.f, bias = 0.f;
    bool key = false;
    const int end = (int)((long long)all * (split + 1) / a.splits);
    int i = (int)((long long)all * split / a.splits);
    auto fetch = [&](int i) __attribute__((always_inline)) {  // pair i: sample i % B of head i / B
        const int ih = uniform(i / a.B), b = uniform(i - ih * a.B);
        const HeadBuf qh = HeadBuf::of<T, D>(a.q, b, ih, a.Lq), kh = HeadBuf::of<T, D>(a.k, b, ih, a.Lk);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int r = (256 * n + tid) / TL::CPR, c = (256 * n + tid) % TL::CPR;
            x[n].load(qh.r, qh.at(q0, qh.at(r, 8 * c * (int)sizeof(T))));
            y[n].load(kh.r, kh.at(k0, kh.at(r, 8 * c * (int)sizeof(T))));
        }
        key = key_there(a, b, k0 + l);
        lse = q < a.Lq ? a.lse[((size_t)b * a.H + ih) * a.Lq + q] : __builtin_inff();
        bias = bias_weight<T>(a, bucket, ih);
    };
    if (i < end) fetch(i);
    for (; i < end; ++i) {
        const unsigned long long there = __ballot(key);
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int r = (256 * n + tid) / TL::CPR, c = (256 * n + tid) % TL::CPR, s = r >> 5;
            x[n].template store<D, true>(lds + s * TL::BYTES, r & 31, c, true);
            if (there == ~0ull) y[n].template store<D, true>(lds + (2 + s) * TL::BYTES, r & 31, c, true);
            else y[n].template store<D, false>(lds + (2 + s) * TL::BYTES, r & 31, c, (there >> r) & 1u);
        }
        if (tid < 127) tab[tid] = bias;
        const float row = lse;
        __syncthreads();
        if (i + 1 < end) fetch(i + 1);
        const unsigned word = (unsigned)(there >> kw);
        if (word == 0) continue;
        const typename TL::Row kr = TL::rows(lds + (2 + (w & 1)) * TL::BYTES, at), qr = TL::rows(lds + (w >> 1) * TL::BYTES, at);
        const f32x16 s = TL::feat(kr, qr);  // rows: keys, lanes: queries
        float t[16];
        if (far) {
            const float add = tab[0] - row;
#pragma unroll
            for (int r = 0; r < 16; ++r) t[r] = fmaf(s[r], c2, add);
        } else {
            const float* bias_at = tab + 63 + kw - qw - li + 4 * h;
#pragma unroll
            for (int r = 0; r < 16; ++r) t[r] = fmaf(s[r], c2, bias_at[8 * (r >> 2) + (r & 3)] - row);
        }
        if (word == ~0u) {
#pragma unroll
            for (int r = 0; r < 16; ++r) sum[r] += __builtin_amdgcn_exp2f(t[r]);
        } else {
            const unsigned mine = word >> (4 * h);
#pragma unroll
            for (int r = 0; r < 16; ++r) sum[r] += (mine >> (8 * (r >> 2) + (r & 3))) & 1u ? __builtin_amdgcn_exp2f(t[r]) : 0.f;
        }
    }
    // queries to the rows
    __syncthreads();
    float* map = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int r = 0; r < 16; ++r) map[(qw + li) * 65 + kw + acc_row(r, h)] = sum[r];
    __syncthreads();
    const float inv = a.splits > 1 ? 1.f : 1.f / all;
    float* out = a.splits > 1 ? a.part + (size_t)split * a.Lq * a.Lk : a.mean;
    if (k0 + l < a.Lk)
        for (int r = w; r < min(64, a.Lq - q0); r += 4) out[(size_t)(q0 + r) * a.Lk + k0 + l] = map[r * 65 + l] * inv;
}
// The pieces' maps, in their order.
__global__ __launch_bounds__(256) void bias_mean_merge_kernel(const float* __restrict__ part, float* __restrict__ mean, long long n,
                                                              int splits, float inv) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        float s = part[i];
        for (int k = 1; k < splits; ++k) s += part[k * n + i];
        mean[i] = s * inv;
    }
}

}  // namespace spion

// Attention with a learned bias by buckets of relative position: no counterpart in the reference (its encoder knows positions
// only from embeddings, models/model_transformer.py:17-52).  With t_ij = (q_i . k_j / sqrt(d) + w[bucket(j - i - off)]) log2(e)
//   forward   P_ij = exp2(t_ij - lse_i),  O = P V
//   backward  dP = dO V^T,  D_i = sum_j P_ij dP_ij,  dS = P (dP - D),  dQ = dS K / sqrt(d),  dK = dS^T Q / sqrt(d),  dV = P^T dO,
//             dw[k] = sum of dS over the pairs of bucket k
// P is never written: the forward leaves lse, the backward forms P again.  Keys whose mask is 0 are left out; with a block
// pattern the keys off the pattern count with a logit of 0, as in models/block_attn.cu:70-72.
//
// The kernels here give a work-group one strip of 32 rows, which is the lane index of every accumulator, and its four wavefronts
// every fourth tile of the strip's list; each stages its tiles in its own part of LDS, so nothing waits for a barrier inside
// the walk, and long strips (a global block row, a single query over a long sample) are shared by four wavefronts and, in the
// forward, by several work-groups.
// Small calls are bound by the latency of a strip's steps (table, list, tiles, the wavefronts' merge): 64 heads, one query over 2048
// padded keys, bf16: 9.6 us and 3.8 for the merge, 33 MB that a copy moves in 6.6; 16 fp32 heads of 1024, d = 32: 27, 33 and 43 us.
#pragma once
#include "bias_tile.h"

namespace spion {

constexpr float BIAS_LAZY = 8.f;  // the running maximum is raised only when a tile exceeds it by 2^8

// floats a piece of a forward strip leaves for the merge: the unscaled sums, maxima, denominators, keys of the pattern
template <int D>
constexpr int bias_slot() { return 32 * D + 96; }

__device__ __forceinline__ int key_bit(unsigned word, int key) { return (word >> key) & 1u; }

// t[r] = logits (log2 domain) of a tile whose keys are the accumulator rows, query on the lane.  One number for the bias of a
// tile far from the strip; NEG: keys that are left out get -infinity.
template <bool MASKED>
__device__ __forceinline__ void logits_of(const f32x16& s, float c2, const float* tab, int R, int rel0, int li, int h,
                                          unsigned word, float (&t)[16]) {
    if (rel0 + 31 > -R && rel0 - 31 < R) {
        const float* at = tab + rel0 + R + BIAS_PAD - li + 4 * h;
#pragma unroll
        for (int r = 0; r < 16; ++r) t[r] = fmaf(s[r], c2, at[8 * (r >> 2) + (r & 3)]);
    } else {
        const float c = tab[rel0 > 0 ? 2 * (R + BIAS_PAD) : 0];
#pragma unroll
        for (int r = 0; r < 16; ++r) t[r] = fmaf(s[r], c2, c);
    }
    if (MASKED) {
        const unsigned mine = word >> (4 * h);
#pragma unroll
        for (int r = 0; r < 16; ++r) t[r] = (mine >> (8 * (r >> 2) + (r & 3))) & 1u ? t[r] : -__builtin_inff();
    }
}

// Work-group -> (sample, head, strip, piece).  The hardware deals work-groups round-robin over the XCDs; the strips of a head follow
// each other on one of them, whose L2 then holds its K and V, and the heads go round-robin, so that every XCD has heads of
// every sample: with key masks samples differ in length (consecutive heads on an XCD instead: 8 heads each of 16 samples of
// 1024 to 2048 tokens take 803 us a step against 753).  What is left of eight heads is spread evenly.
struct BiasItem {
    int b, h, bh, strip, split;
    __device__ __forceinline__ BiasItem(const BiasCall& a, int total) {
        const int each = a.strips * a.splits, whole = a.B * a.H / 8 * 8 * each;  // work-groups of a head, of the whole rounds
        int i = blockIdx.x;
        if (i < whole) {
            const int n = i / 8;
            i = (n / each * 8 + i % 8) * each + n % each;
        } else {
            i = whole + xcd_remap(i - whole, total - whole);
        }
        split = i % a.splits;
        i /= a.splits;
        strip = i % a.strips;
        bh = i / a.strips;
        b = bh / a.H;
        h = bh - b * a.H;
    }
    // wavefront w's slot in a launch with strips of 128: the pieces of 32 rows lie next to each other
    __device__ __forceinline__ size_t slot(const BiasCall& a, int w) const {
        return ((size_t)bh * a.strips32 + strip * 4 + w) * a.splits + split;
    }
};

// Wavefronts a SIMD that the registers are for.  fp32 heads of 64 features: one.  Strips of 32 have one work-group's tiles in a CU's
// LDS (98 KB); the backward passes over shared stages take 56 to 93 KB, which mostly leaves room for two, but 320 and 350 registers.
// (The bf16 column pass of strips of 32 at d = 64 has all of its 256 registers in use and spills 44 bytes a lane.)
template <class T, int D>
constexpr int bias_waves() { return sizeof(T) == 4 && D == 64 ? 1 : 2; }

template <class T, int D>
constexpr int bias_tiles_bytes() {
    const int tiles = 4 * 2 * BiasTile<T, D>::BYTES, merge = merge_floats<D>() * 4;
    return tiles > merge ? tiles : merge;
}

// Eighth j of row i of a tensor
template <class T, int D>
__device__ __forceinline__ void store_eighth(const HeadsAt& t, int b, int h, int i, int j, const float (&x)[D / 8]) {
    store_values<T, D / 8>(const_cast<char*>(t.head(b, h)) + i * t.row + j * (D / 8) * sizeof(T), x);
}

// -------------------------------------------------------------------------------------------------
// Forward
// -------------------------------------------------------------------------------------------------
template <class T, int D>
__global__ __launch_bounds__(256, (bias_waves<T, D>())) void bias_forward_kernel(BiasCall a) {
    typedef BiasTile<T, D> TL;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float* tab = reinterpret_cast<float*>(lds + bias_tiles_bytes<T, D>());
    ScanLds& sc = *reinterpret_cast<ScanLds*>(tab + bias_floats(a.R));
    const int tid = threadIdx.x, w = uniform(tid >> 6), l = tid & 63, li = l & 31, h = l >> 5;
    const BiasItem it(a, gridDim.x);
    fill_bias<T>(a, it.h, tab, tid);
    const int q0 = it.strip * 32;
    const typename TL::Row q = TL::load(a.q.head(it.b, it.h) + min(q0 + li, a.Lq - 1) * a.q.row, h, q0 + li < a.Lq);
    const HeadBuf kh = HeadBuf::of<T, D>(a.k, it.b, it.h, a.Lk), vh = HeadBuf::of<T, D>(a.v, it.b, it.h, a.Lk);
    const typename TL::At at = TL::at(l);
    char* tk = lds + w * 2 * TL::BYTES;
    char* tv = tk + TL::BYTES;
    const float c2 = a.scale * LOG2E;
    const int qpos = q0 + a.off;
    q.settled();

    f32x16 o[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) o[c] = splat16(0.f);
    float m = -__builtin_inff(), z = 0.f;
    int in_pattern = 0;
    const int tiles = (a.Lk + 31) / 32;
    const int t0 = it.split * a.per_split, t1 = min(tiles, t0 + a.per_split);
    for (int first = t0; first < t1; first += CHUNK) {
        const int n = scan_chunk<true>(a, sc, it.b, it.strip, first, min(CHUNK, t1 - first), tid, in_pattern);
        TileInFlight<T, D> fk, fv;
        auto fetch = [&](int i) __attribute__((always_inline)) {
            const int j = (first + uniform(sc.list[i])) * 32;
            fk.load(kh, j, l);
            fv.load(vh, j, l);
        };
        if (w < n) fetch(w);
        for (int i = w; i < n; i += 4) {
            const int tile = uniform(sc.list[i]);
            const unsigned word = uniform(sc.words[tile]);
            wave_lds_order();
            fk.store(tk, word, l);
            fv.store(tv, word, l);
            wave_lds_order();
            if (i + 4 < n) fetch(i + 4);
            const typename TL::Row kr = TL::rows(tk, at);
            typename TL::Columns vt;
            if (TL::EARLY) vt = TL::columns(tv, at);
            issue_order();
            const f32x16 s = TL::feat(kr, q);
            float t[16];
            const int rel0 = (first + tile) * 32 - qpos;
            if (word == ~0u) logits_of<false>(s, c2, tab, a.R, rel0, li, h, word, t);
            else logits_of<true>(s, c2, tab, a.R, rel0, li, h, word, t);
            float mt = t[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) mt = fmaxf(mt, t[r]);
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
            const float base = m == -__builtin_inff() ? 0.f : m;
            float p[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                p[r] = __builtin_amdgcn_exp2f(t[r] - base);
                z += p[r];
            }
            if (!TL::EARLY) vt = TL::columns(tv, at);
            TL::add_t(vt, p, o);
        }
    }
    // the four wavefronts' parts
    z = half_swap_sum(z);
    if (h == 0) {
        sc.ml[w][0][li] = m;
        sc.ml[w][1][li] = z;
    }
    __syncthreads();
    float M = sc.ml[0][0][li];
#pragma unroll
    for (int k = 1; k < 4; ++k) M = fmaxf(M, sc.ml[k][0][li]);
    const float base = M == -__builtin_inff() ? 0.f : M;
    float Z = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) Z += sc.ml[k][1][li] * __builtin_amdgcn_exp2f(sc.ml[k][0][li] - base);
    const float f = __builtin_amdgcn_exp2f(m - base);
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[c][r] *= f;
    float x[D / 8];
    merge_waves<D>(o, reinterpret_cast<float*>(lds), tid, x);
    const int row = tid >> 3, j = tid & 7;
    if (a.splits > 1) {
        float* slot = a.part + (size_t)((it.bh * (size_t)a.strips + it.strip) * a.splits + it.split) * bias_slot<D>();
        // (rows behind the last query are not read again: of a single query's pieces 0.3 KB are written, not 8.6)
        if (q0 + row < a.Lq) store_values<float, D / 8>(reinterpret_cast<char*>(slot + row * D + j * (D / 8)), x);
        if (w == 0 && h == 0) {
            slot[32 * D + li] = M;
            slot[32 * D + 32 + li] = Z;
            slot[32 * D + 64 + li] = __builtin_bit_cast(float, in_pattern);
        }
        return;
    }
    if (w == 0 && h == 0) {
        const int off = a.mat ? a.Lk - in_pattern : 0;  // keys off the pattern: a logit of 0 each
        float scale = 1.f;
        if (off > 0) {
            const float up = fmaxf(M, 0.f);
            scale = __builtin_amdgcn_exp2f(M - up);
            Z = Z * scale + off * __builtin_amdgcn_exp2f(-up);
            M = up;
        }
        sc.row[li] = Z == 0.f ? 0.f : scale / Z;
        if (q0 + li < a.Lq)
            a.lse[(size_t)it.bh * a.Lq + q0 + li] = Z == 0.f ? __builtin_inff() : M + __builtin_amdgcn_logf(Z);
    }
    __syncthreads();
    if (q0 + row < a.Lq) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) x[i] *= sc.row[row];
        store_eighth<T, D>(a.o, it.b, it.h, q0 + row, j, x);
    }
}

// The pieces of a strip, in their order; eight pieces' loads are in flight together (there is little else in this launch than the
// two waits for them).
template <class T, int D>
__global__ __launch_bounds__(256) void bias_merge_kernel(BiasCall a) {
    const int tid = threadIdx.x, row = tid >> 3, j = tid & 7;
    const int strip = blockIdx.x % a.strips32, bh = blockIdx.x / a.strips32, b = bh / a.H, ih = bh - b * a.H;
    const int q = strip * 32 + row;
    if (q >= a.Lq) return;
    const float* slot = a.part + (size_t)blockIdx.x * a.splits * bias_slot<D>();
    float M = -__builtin_inff();
    int in_pattern = 0;
#pragma unroll 8
    for (int k = 0; k < a.splits; ++k) {
        M = fmaxf(M, slot[k * bias_slot<D>() + 32 * D + row]);
        in_pattern += __builtin_bit_cast(int, slot[k * bias_slot<D>() + 32 * D + 64 + row]);
    }
    const int off = a.mat ? a.Lk - in_pattern : 0;
    if (off > 0) M = fmaxf(M, 0.f);
    const float base = M == -__builtin_inff() ? 0.f : M;
    float Z = off > 0 ? off * __builtin_amdgcn_exp2f(-base) : 0.f, x[D / 8];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) x[i] = 0.f;
#pragma unroll 8
    for (int k = 0; k < a.splits; ++k) {
        const float* s = slot + k * bias_slot<D>();
        const float f = __builtin_amdgcn_exp2f(s[32 * D + row] - base);
        Z += s[32 * D + 32 + row] * f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(s + row * D + j * (D / 8) + 4 * i);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * i + e] += v[e] * f;
        }
    }
    const float inv = Z == 0.f ? 0.f : 1.f / Z;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) x[i] *= inv;
    store_eighth<T, D>(a.o, b, ih, q, j, x);
    if (j == 0) a.lse[(size_t)bh * a.Lq + q] = Z == 0.f ? __builtin_inff() : M + __builtin_amdgcn_logf(Z);
}

// -------------------------------------------------------------------------------------------------
// Backward, strips of queries: dQ and D
// -------------------------------------------------------------------------------------------------
// D = dO . O to begin with, from the output as it was rounded (and summed with rounded weights): good for dQ, whose own rounding is
// larger.  The strip's sum of P (dP - dO.O) then gives what is left to D = sum_j P_ij dP_ij of the P that the backward itself forms,
// and the column pass has that.  (The table's gradient adds up P (dP - D) over thousands of rows whose terms nearly cancel:
// with dO.O for D the buckets of far keys come out wrong by 0.8 %, 28 heads of 2923 tokens in bf16, 8 buckets, against 0.16 % of
// rounding at the end.)
//
// With rest = off * exp2(-lse), what keys off the pattern have of the row's probabilities, and S = 1 - rest: the strip's `sum` is
// sum_j P (dP - dO.O), and D = S dO.O + sum.  In fp32 that is not all.  The matrix units' products come out low by some b (2.8e-8 in
// the mean at d = 32), while dO.O, added up by the vector units, has none of it: sum = rest dO.O + S b, and D = dO.O + S b.  But
// every dP of the column pass has the whole b, so D is to have it as well: D = dO.O + (sum - rest dO.O) / S.  (S b left the far
// buckets off by b S (1 - S) a row, all of one sign: 2.7e-6 of the table's gradient, 6 heads of 2994, a quarter of the blocks.)
// bf16 outputs, and dO.O with them, are rounded by far more than b.
template <class T>
__device__ __forceinline__ float exact_d(float delta, float sum, float lse, int off) {
    const float rest = off > 0 ? off * __builtin_amdgcn_exp2f(-lse) : 0.f, S = 1.f - rest;
    if (sizeof(T) == 4 && rest > 0.f && S > 0.f) return delta + fmaf(-delta, rest, sum) / S;
    return fmaf(delta, S, sum);
}

template <class T, int D>
__global__ __launch_bounds__(256, (bias_waves<T, D>())) void bias_backward_row_kernel(BiasCall a) {
    typedef BiasTile<T, D> TL;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float* tab = reinterpret_cast<float*>(lds + bias_tiles_bytes<T, D>());
    ScanLds& sc = *reinterpret_cast<ScanLds*>(tab + bias_floats(a.R));
    const int tid = threadIdx.x, w = uniform(tid >> 6), l = tid & 63, li = l & 31, h = l >> 5;
    const BiasItem it(a, gridDim.x);
    fill_bias<T>(a, it.h, tab, tid);
    const int q0 = it.strip * 32, qi = min(q0 + li, a.Lq - 1);
    const bool there = q0 + li < a.Lq;
    const typename TL::Row q = TL::load(a.q.head(it.b, it.h) + qi * a.q.row, h, there);
    const typename TL::Row go = TL::load(a.dout.head(it.b, it.h) + qi * a.dout.row, h, there);
    const size_t stat = (size_t)it.bh * a.Lq + qi;
    const float lse = there ? a.lse[stat] : __builtin_inff();
    const float delta = half_swap_sum(TL::dot(go, TL::load(a.o.head(it.b, it.h) + qi * a.o.row, h, there)));
    const HeadBuf kh = HeadBuf::of<T, D>(a.k, it.b, it.h, a.Lk), vh = HeadBuf::of<T, D>(a.v, it.b, it.h, a.Lk);
    const typename TL::At at = TL::at(l);
    char* tk = lds + w * 2 * TL::BYTES;
    char* tv = tk + TL::BYTES;
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
    const int tiles = (a.Lk + 31) / 32;
    for (int first = 0; first < tiles; first += CHUNK) {
        const int n = scan_chunk<true>(a, sc, it.b, it.strip, first, min(CHUNK, tiles - first), tid, in_pattern);
        TileInFlight<T, D> fk, fv;
        auto fetch = [&](int i) __attribute__((always_inline)) {
            const int j = (first + uniform(sc.list[i])) * 32;
            fk.load(kh, j, l);
            fv.load(vh, j, l);
        };
        if (w < n) fetch(w);
        for (int i = w; i < n; i += 4) {
            const int tile = uniform(sc.list[i]);
            const unsigned word = uniform(sc.words[tile]);
            wave_lds_order();
            fk.store(tk, word, l);
            fv.store(tv, word, l);
            wave_lds_order();
            if (i + 4 < n) fetch(i + 4);
            const typename TL::Row kr = TL::rows(tk, at), vr = TL::rows(tv, at);
            typename TL::Columns kt;
            if (TL::EARLY) kt = TL::columns(tk, at);
            issue_order();
            const f32x16 s = TL::feat(kr, q);
            const f32x16 dp = TL::feat(vr, go, minus);  // dP - D
            float t[16];
            const int rel0 = (first + tile) * 32 - qpos;
            if (word == ~0u) logits_of<false>(s, c2, tab, a.R, rel0, li, h, word, t);
            else logits_of<true>(s, c2, tab, a.R, rel0, li, h, word, t);
            float ds[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                ds[r] = __builtin_amdgcn_exp2f(t[r] - lse) * dp[r];
                sum += ds[r];
            }
            if (!TL::EARLY) kt = TL::columns(tk, at);
            TL::add_t(kt, ds, dq);
        }
    }
    sum = half_swap_sum(sum);
    if (h == 0) sc.ml[w][0][li] = sum;
    __syncthreads();  // the tiles are done with
    if (w == 0 && h == 0 && there) {
        const float all = (sc.ml[0][0][li] + sc.ml[1][0][li]) + (sc.ml[2][0][li] + sc.ml[3][0][li]);
        a.delta[stat] = exact_d<T>(delta, all, lse, a.mat ? a.Lk - in_pattern : 0);
    }
    float x[D / 8];
    merge_waves<D>(dq, reinterpret_cast<float*>(lds), tid, x);
    const int row = tid >> 3, j = tid & 7;
    if (q0 + row < a.Lq) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) x[i] *= a.scale;
        store_eighth<T, D>(a.dq, it.b, it.h, q0 + row, j, x);
    }
}

// -------------------------------------------------------------------------------------------------
// Backward, strips of keys: dK, dV and the table's gradient
// -------------------------------------------------------------------------------------------------
// The strip's keys are the lanes: what a key that is left out holds reaches its own lane only, whose results are zeros.
//
// The table's gradient: dS summed by difference.  Of a tile outside (-R, R) only its sum is needed, which stays in a register.  A
// tile that touches the range is summed along its diagonals: the wavefront writes 16 of its rows to LDS so that a diagonal is
// a column, four rows to a 16-byte piece, reads the columns back, a lane each, and adds their sums to its histogram of differences
// (an LDS atomic per register and lane instead took a third of the kernel that had it: 735 us against 490 without any sums,
// 128 padded heads of 2048, where a seventh of the tiles touch the range).  Every histogram is added to by one wavefront in
// program order, no two lanes of an instruction meet: the sums come out the same each time.  The histograms of a strip are added
// up, folded into buckets and left in the workspace, [strips][buckets] for every head.
constexpr int BIAS_HISTS = 4, DIAG_COLS = 48, DIAG_FLOATS = 4 * DIAG_COLS * 4;
// ds: rows are queries, lanes keys; hist: at difference rel0 (of the tile's first key and query); buf: the wavefront's, places that
// are never written are zeros
__device__ __forceinline__ void add_diagonals(float* buf, float* hist, const float (&ds)[16], int li, int h) {
    const int l = li + 32 * h;
    float* mine = buf + (h * DIAG_COLS + li - 4 * h + 15) * 4;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        wave_lds_order();
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) mine[(2 * g * DIAG_COLS - 8 * g - e) * 4 + e] = ds[8 * half + 4 * g + e];
        wave_lds_order();
        if (l < DIAG_COLS - 1) {
            f32x4 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const f32x4*>(buf + (k * DIAG_COLS + l) * 4);
            const f32x4 s = (v[0] + v[1]) + (v[2] + v[3]);
            __hip_atomic_fetch_add(hist - 16 * half - 15 + l, (s[0] + s[1]) + (s[2] + s[3]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
    }
}
// The wavefronts' histograms into buckets, in a fixed order whatever the map is.  Neighbouring entries mostly share their bucket: a
// wavefront adds up a block of 64 entries by runs of one bucket (a scan that stops where a run begins) and leaves the runs' sums
// and buckets, in order, where the block was.  Then eight threads to a bucket go through the runs, each through every eighth
// block's.  (Every entry looked at for every bucket, against this, in a column pass with nothing in its pattern, 16 heads of 8192 in
// strips of 64, us: R = 16 39 / 44, R = 128 47 / 45, R = 1024 183 / 119.)  LDS behind a barrier; runs: an int to a block.
__device__ __forceinline__ void fold_hists(float* hist, unsigned short* bucket, int* runs, int entries, int buckets, int tid, float* part) {
    const int w = uniform(tid >> 6), l = tid & 63, blocks = (entries + 63) / 64;
    for (int b = w; b < blocks; b += 4) {
        const int i = b * 64 + l;
        const bool in = i < entries;
        const int k = in ? bucket[i] : -1;
        float s = in ? (hist[i] + hist[entries + i]) + (hist[2 * entries + i] + hist[3 * entries + i]) : 0.f;
        const int before = __shfl_up(k, 1, 64);
        const unsigned long long begins = __ballot(l == 0 || before != k), upto = begins & (~0ull >> (63 - l));
        const int from = 63 - __clzll(upto);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const float x = __shfl_up(s, o, 64);
            if (l - o >= from) s += x;
        }
        const bool last = in && (l == 63 || ((begins >> 1) >> l) & 1);
        const unsigned long long ends = __ballot(last);
        const int at = b * 64 + __popcll(ends & ((1ull << l) - 1));  // (no further than i, which this wavefront has read)
        wave_lds_order();
        if (last) {
            hist[at] = s;
            bucket[at] = (unsigned short)k;
        }
        if (l == 0) runs[b] = __popcll(ends);
    }
    __syncthreads();
    for (int k0 = 0; k0 < buckets; k0 += 32) {
        const int k = k0 + (tid >> 3);
        float s = 0.f;
        for (int b = tid & 7; b < blocks; b += 8) {
            const int n = runs[b];
#pragma unroll 4
            for (int i = b * 64; i < b * 64 + n; ++i) s += bucket[i] == k ? hist[i] : 0.f;
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) s += __shfl_xor(s, o, 64);
        if (k < buckets && (tid & 7) == 0) part[k] = s;
    }
}
// LDS of the kernels that make the table's gradient, behind the scan's: the wavefronts' diagonals, their histograms, the entries'
// buckets
struct HistLds {
    float *diag, *hist;
    unsigned short* bucket;
    __device__ __forceinline__ HistLds(ScanLds& sc, int R)
        : diag(reinterpret_cast<float*>(&sc + 1)), hist(diag + BIAS_HISTS * DIAG_FLOATS),
          bucket(reinterpret_cast<unsigned short*>(hist + BIAS_HISTS * bias_entries(R))) {}
    __device__ __forceinline__ void clear(int R, int tid) {
        for (int i = tid; i < BIAS_HISTS * (DIAG_FLOATS + bias_entries(R)); i += 256) diag[i] = 0.f;
    }
    __host__ __device__ static int bytes(int R) { return BIAS_HISTS * (DIAG_FLOATS + bias_entries(R)) * 4 + ((bias_entries(R) * 2 + 15) & ~15); }
};
// A wavefront's sums: dS of a tile, whose lanes are keys of which `key` says whether they take part
struct DifferenceSums {
    float *hist, *diag;
    int R;
    bool key, some_out;  // some_out: a key of the strip is left out
    float behind = 0.f, ahead = 0.f;
    __device__ __forceinline__ DifferenceSums(const HistLds& hl, int w, int R_, bool key_)
        : hist(hl.hist + w * bias_entries(R_) + R_ + BIAS_PAD), diag(hl.diag + w * DIAG_FLOATS), R(R_), key(key_), some_out(!__all(key_)) {}
    __device__ __forceinline__ bool touches(int rel0) const { return rel0 + 31 > -R && rel0 - 31 < R; }
    __device__ __forceinline__ void near(int rel0, const float (&ds)[16], int li, int h) {
        if (some_out) {
            float kept[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) kept[r] = key ? ds[r] : 0.f;
            add_diagonals(diag, hist + rel0, kept, li, h);
        } else {
            add_diagonals(diag, hist + rel0, ds, li, h);
        }
    }
    __device__ __forceinline__ void far(int rel0, const float (&ds)[16]) {
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += ds[r];
        if (rel0 > 0) ahead += sum;
        else behind += sum;
    }
    __device__ __forceinline__ void finish(int l) {
        const float b = wave_sum(key ? behind : 0.f), f = wave_sum(key ? ahead : 0.f);
        if (l == 0) {
            hist[-R - BIAS_PAD] += b;
            hist[R + BIAS_PAD] += f;
        }
    }
};

template <class T, int D>
__global__ __launch_bounds__(256, (bias_waves<T, D>())) void bias_backward_col_kernel(BiasCall a) {
    typedef BiasTile<T, D> TL;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float* tab = reinterpret_cast<float*>(lds + bias_tiles_bytes<T, D>());
    ScanLds& sc = *reinterpret_cast<ScanLds*>(tab + bias_floats(a.R));
    HistLds hl(sc, a.R);
    const int tid = threadIdx.x, w = uniform(tid >> 6), l = tid & 63, li = l & 31, h = l >> 5;
    const BiasItem it(a, gridDim.x);
    fill_bias<T>(a, it.h, tab, tid, hl.bucket);
    hl.clear(a.R, tid);
    const int k0 = it.strip * 32, ki = min(k0 + li, a.Lk - 1);
    const typename TL::Row k = TL::load(a.k.head(it.b, it.h) + ki * a.k.row, h, k0 + li < a.Lk);
    const typename TL::Row v = TL::load(a.v.head(it.b, it.h) + ki * a.v.row, h, k0 + li < a.Lk);
    const bool key = key_there(a, it.b, k0 + li);
    const unsigned keys = (unsigned)__ballot(key);
    DifferenceSums sums(hl, w, a.R, key);
    const HeadBuf qh = HeadBuf::of<T, D>(a.q, it.b, it.h, a.Lq), gh = HeadBuf::of<T, D>(a.dout, it.b, it.h, a.Lq);
    const float *lseh = a.lse + (size_t)it.bh * a.Lq, *deltah = a.delta + (size_t)it.bh * a.Lq;
    const typename TL::At at = TL::at(l);
    char* tq = lds + w * 2 * TL::BYTES;
    char* tg = tq + TL::BYTES;
    float* stats = sc.ml[w][0];  // lse of the tile's 32 queries, then their -D
    const float c2 = a.scale * LOG2E;
    k.settled();
    v.settled();

    f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) dk[c] = dv[c] = splat16(0.f);
    int in_pattern = 0;
    const int tiles = keys == 0 ? 0 : (a.Lq + 31) / 32;  // the same in every thread
    for (int first = 0; first < tiles; first += CHUNK) {
        const int n = scan_chunk<false>(a, sc, it.b, it.strip, first, min(CHUNK, tiles - first), tid, in_pattern);
        TileInFlight<T, D> fq, fg;
        float st = 0.f;
        auto fetch = [&](int i) __attribute__((always_inline)) {
            const int r = (first + uniform(sc.list[i])) * 32;
            fq.load(qh, r, l);
            fg.load(gh, r, l);
            st = r + li < a.Lq ? (h ? -deltah[r + li] : lseh[r + li]) : (h ? 0.f : __builtin_inff());
        };
        if (w < n) fetch(w);
        for (int i = w; i < n; i += 4) {
            const int tile = uniform(sc.list[i]);
            const int r0 = (first + tile) * 32;
            const unsigned word = tail_word(a.Lq - r0);
            wave_lds_order();
            fq.store(tq, word, l);
            fg.store(tg, word, l);
            stats[l] = st;
            wave_lds_order();
            if (i + 4 < n) fetch(i + 4);
            f32x16 dp;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 d = *reinterpret_cast<const f32x4*>(stats + 32 + 8 * g + 4 * h);
#pragma unroll
                for (int j = 0; j < 4; ++j) dp[4 * g + j] = d[j];
            }
            const typename TL::Row qr = TL::rows(tq, at), gr = TL::rows(tg, at);
            typename TL::Columns qt, gt;
            if (TL::EARLY) qt = TL::columns(tq, at), gt = TL::columns(tg, at);
            issue_order();
            const f32x16 s = TL::feat(qr, k);
            dp = TL::feat(gr, v, dp);  // dP - D
            const int rel0 = k0 - r0 - a.off;  // of the tile's corner: lane li, row r has rel0 + li - r
            const bool near = sums.touches(rel0);
            float p[16];
            if (near) {
                const float* bias = tab + rel0 + a.R + BIAS_PAD + li - 4 * h;
#pragma unroll
                for (int r = 0; r < 16; ++r) p[r] = fmaf(s[r], c2, bias[-(8 * (r >> 2) + (r & 3))]);
            } else {
                const float c = tab[rel0 > 0 ? 2 * (a.R + BIAS_PAD) : 0];
#pragma unroll
                for (int r = 0; r < 16; ++r) p[r] = fmaf(s[r], c2, c);
            }
            float ds[16];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 e = *reinterpret_cast<const f32x4*>(stats + 8 * g + 4 * h);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    p[4 * g + j] = __builtin_amdgcn_exp2f(p[4 * g + j] - e[j]);
                    ds[4 * g + j] = p[4 * g + j] * dp[4 * g + j];
                }
            }
            if (near) sums.near(rel0, ds, li, h);
            else sums.far(rel0, ds);
            if (!TL::EARLY) gt = TL::columns(tg, at);
            TL::add_t(gt, p, dv);
            if (!TL::EARLY) qt = TL::columns(tq, at);
            TL::add_t(qt, ds, dk);
        }
    }
    if (keys == 0) __syncthreads();  // the tables are there (a scan has seen to it otherwise)
    sums.finish(l);
    __syncthreads();
    const int row = tid >> 3, j = tid & 7;
    const bool keep = key_bit(keys, row);
    float x[D / 8];
    merge_waves<D>(dv, reinterpret_cast<float*>(lds), tid, x);
    if (k0 + row < a.Lk) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) x[i] = keep ? x[i] : 0.f;
        store_eighth<T, D>(a.dv, it.b, it.h, k0 + row, j, x);
    }
    __syncthreads();
    merge_waves<D>(dk, reinterpret_cast<float*>(lds), tid, x);
    if (k0 + row < a.Lk) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) x[i] = keep ? x[i] * a.scale : 0.f;
        store_eighth<T, D>(a.dk, it.b, it.h, k0 + row, j, x);
    }
    fold_hists(hl.hist, hl.bucket, reinterpret_cast<int*>(hl.diag), bias_entries(a.R), a.buckets, tid, a.tables + ((size_t)it.bh * a.strips + it.strip) * a.buckets);
}

// dw[k][h]: the strips' pieces of all samples, 256 partial sums in a fixed order.
template <class T>
__global__ __launch_bounds__(256) void bias_table_kernel(BiasCall a, T* __restrict__ dw) {
    __shared__ float red[4];
    const int k = blockIdx.x % a.buckets, h = blockIdx.x / a.buckets, tid = threadIdx.x;
    const int each = a.strips * a.splits, n = a.B * each;
    float s = 0.f;
#pragma unroll 4
    for (int i = tid; i < n; i += 256) {
        const int b = i / each, piece = i - b * each;
        s += a.tables[(((size_t)b * a.H + h) * each + piece) * a.buckets + k];
    }
    s = wave_sum(s);
    if ((tid & 63) == 0) red[tid >> 6] = s;
    __syncthreads();
    if (tid == 0) dw[(size_t)k * a.H + h] = (T)(red[0] + red[1] + red[2] + red[3]);
}

}  // namespace spion

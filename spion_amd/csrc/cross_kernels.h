// Attention of queries to keys of another length (no counterpart in the reference, whose attention is an encoder's own,
// models/attention.py:79-103): cross attention, with heads of keys that several heads of queries share.
// With t_ij = (q_i . k_j) log2(e) / sqrt(d) over the keys that take part
//   forward   P_ij = exp2(t_ij - lse_i),  O = P V
//   backward  dP = dO V^T,  D_i = dO_i . O_i,  dS = P (dP - D),  dQ = dS K / sqrt(d),  dK = dS^T Q / sqrt(d),  dV = P^T dO
// No position enters, so the queries of the heads that share a head of keys are rows of one problem: row r of such a group is query
// r % Lq of its head r / Lq.  K and V of a group are then read once for all of them, a single token of four heads is four rows of
// one strip, and dK and dV are summed over the group by the products themselves.
// P is never written: the forward leaves lse, and the backward, in a pass over rows (dQ) and one over keys (dK, dV), forms P again.
// Long calls are bound by issue and power (matrix units 41 to 48 % busy at 1.9 GHz; TFLOP/s of forward / rows / keys, bf16: d = 32 530 / 740 / 735, d = 64
// 755 / 910 / 862, d = 128 940 / 1080 / 950; fp32, six bf16 products counted as one: 163 to 197), calls of few rows by memory (one token of
// 4 x 16 heads over 4, 32768 keys, d = 128: 268 MB in 46 us), small ones by the latency of a strip: some 0.5 us a step, 2 to 3 us to start and end.
#pragma once
#include "bias_tile.h"

#include <type_traits>

namespace spion {

struct CrossCall {
    HeadsAt q, k, v, o, dout, dq, dk, dv;
    const void* mask;  // [B][Lk]: null, float (0 = left out) or bytes
    float* lse;        // [B * G][rows]: log2 of the softmax denominator, +inf for rows that nothing enters (NaN stays NaN)
    float* delta;      // [B * G][rows]: dO . O
    float* part;       // workspace: the pieces' slots
    int B, G, each, Lq, Lk, rows;  // G heads of keys, each for `each` heads of queries; rows = each * Lq
    unsigned magic;                // r / Lq = r * magic >> shift, for r < 2^31
    int shift;
    int mask_bytes;                  // 4 or 1
    int strips, splits, per_split;   // strips of a head's rows or keys, pieces of the other side, tiles of 32 to a piece
    float scale;
    __device__ __forceinline__ int head_of(int r) const { return each == 1 ? 0 : (int)((unsigned long long)(unsigned)r * magic >> shift); }
    // row r of group g of sample b
    __device__ __forceinline__ const char* row(const HeadsAt& t, int b, int g, int r) const {
        const int n = head_of(r);
        return t.p + b * t.b + (g * (long long)each + n) * t.h + (r - n * Lq) * t.row;
    }
};

// The running maximum is raised only when a tile exceeds it by 2^8: sums stay below 2^8 times the keys, and most tiles have nothing
// to rescale.
constexpr float CROSS_LAZY = 8.f;

// Rows that are staged: a head of keys, or a group of queries.  A head, or a group, lies within 2^31 bytes and its rows 2^24 apart at
// most; rows up to 64 behind the last are asked for (and left out when they are stored to LDS): they read as the last row or as zeros.
template <class T, int D, bool KEYS>
struct CrossSource {
    rsrc_t r;
    unsigned long long first_row;
    unsigned bytes;
    int ld, head;
    const CrossCall& a;
    __device__ __forceinline__ CrossSource(const CrossCall& a, const HeadsAt& t, int b, int g) : ld((int)t.row), head((int)t.h), a(a) {
        const unsigned long long p = reinterpret_cast<unsigned long long>(t.p + b * t.b + (KEYS ? g : g * (long long)a.each) * t.h);
        // (the same in every lane, which the compiler does not see through the divisions that b and g come from)
        first_row = (unsigned)uniform((int)(unsigned)p) | (unsigned long long)(unsigned)uniform((int)(p >> 32)) << 32;
        bytes = (unsigned)((KEYS ? (a.Lk - 1) * t.row : (a.each - 1) * t.h + (a.Lq - 1) * t.row) + D * (int)sizeof(T));
        r = make_rsrc(reinterpret_cast<const void*>(first_row), bytes);
    }
    // whether the rows lie one behind the other
    __device__ __forceinline__ bool linear() const { return KEYS || a.each == 1; }
    __device__ __forceinline__ int at(int first, int row, int byte) const {
        if (linear()) return (int)((unsigned)first * (unsigned)ld + ((unsigned)row * (unsigned)ld + (unsigned)byte));
        const int x = min(first + row, a.rows - 1), n = a.head_of(x);
        return (int)((unsigned)n * (unsigned)head + (unsigned)(x - n * a.Lq) * (unsigned)ld + (unsigned)byte);
    }
};

// The same from row `first` on (an existing one), for loads into LDS: what follows the buffer's end is out of its range, whatever the lane.
template <class S>
__device__ __forceinline__ u32x4 cross_words(const S& s, int first) {
    const unsigned skip = s.linear() ? (unsigned)first * (unsigned)s.ld : 0u;
    const unsigned long long p = s.first_row + skip;
    return u32x4{(unsigned)uniform((int)(unsigned)p), (unsigned)uniform((int)(p >> 32)), (unsigned)uniform((int)(s.bytes - skip)), 0x00020000u};
}
template <class S>
__device__ __forceinline__ int cross_lane(const S& s, int first, int row, int byte) {
    return s.linear() ? row * s.ld + byte : s.at(first, row, byte);
}

// Work-group -> (group, strip, piece): the strips of a group follow each other on one XCD, whose L2 then holds what they share, and
// the groups go round-robin, so that every XCD has groups of every sample (padded ones differ in length).
struct CrossItem {
    int b, g, bg, strip, split;
    __device__ __forceinline__ CrossItem(const CrossCall& a, int total) {
        const int each = a.strips * a.splits, whole = a.B * a.G / 8 * 8 * each;  // work-groups of a group, of the whole rounds
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
        bg = i / a.strips;
        b = bg / a.G;
        g = bg - b * a.G;
    }
    // the piece's slot for 32 rows (or keys), of which the head has `all`
    __device__ __forceinline__ size_t slot(const CrossCall& a, int all, int first) const {
        return ((size_t)bg * ((all + 31) / 32) + first / 32) * a.splits + split;
    }
};

// floats a piece leaves: of the forward the unscaled sums, maxima and denominators, of the row pass dQ, of the column pass dV and dK
template <int D>
constexpr int cross_slot() { return 32 * D + 64; }

// ---------------------------------------------------------------------------------------------------------------------
// Which keys take part
// ---------------------------------------------------------------------------------------------------------------------
// Keys are walked in chunks of CHUNK tiles of 32; with a mask the work-group makes, in LDS, the words of a chunk (which keys of each
// tile take part) and the list of its stages that have any.  The mask is read as it is at the call.
struct CrossLds {
    unsigned words[CHUNK];
    unsigned of[CHUNK];  // the same in the order of the list
    unsigned short list[CHUNK];
    int seg[8];
};
static_assert(sizeof(CrossLds) % 16 == 0, "what follows it is aligned");

__device__ __forceinline__ bool cross_key(const CrossCall& a, int b, int key) {
    if (key >= a.Lk) return false;
    if (a.mask == nullptr) return true;
    const size_t i = (size_t)b * a.Lk + key;
    return a.mask_bytes == 4 ? reinterpret_cast<const float*>(a.mask)[i] != 0.f : reinterpret_cast<const unsigned char*>(a.mask)[i] != 0;
}

// The stages of SUBS tiles among tiles first .. first + count - 1 that have a key: how many; which, in s.list, and their words in s.of.  All 256 threads; LDS that
// they still read must be done with.
template <int SUBS>
__device__ __forceinline__ int cross_scan(const CrossCall& a, CrossLds& s, int b, int first, int count, int tid) {
    const int w = uniform(tid >> 6), l = tid & 63;
    __syncthreads();
    const size_t row = (size_t)b * a.Lk;
    if (a.mask_bytes == 4) mask_words(reinterpret_cast<const float*>(a.mask) + row, s.words, first, (count + 1) / 2, a.Lk, w, l);
    else mask_words(reinterpret_cast<const unsigned char*>(a.mask) + row, s.words, first, (count + 1) / 2, a.Lk, w, l);
    __syncthreads();
    constexpr int ROUNDS = CHUNK / SUBS / 256;
    bool act[ROUNDS];
    unsigned long long votes[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int i = tid + 256 * r;
        unsigned any = i * SUBS < count ? s.words[i * SUBS] : 0u;
        if (SUBS == 2 && i * SUBS + 1 < count) any |= s.words[i * SUBS + 1];
        act[r] = any != 0;
        votes[r] = __ballot(act[r]);
        if (l == 0) s.seg[4 * r + w] = __popcll(votes[r]);
    }
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        int before = 0;
#pragma unroll
        for (int k = 0; k < 4 * ROUNDS; ++k) before += k < 4 * r + w ? s.seg[k] : 0;
        if (!act[r]) continue;
        const int at = before + __popcll(votes[r] & ((1ull << l) - 1)), i = tid + 256 * r;
        s.list[at] = (unsigned short)i;
#pragma unroll
        for (int u = 0; u < SUBS; ++u) s.of[at * SUBS + u] = i * SUBS + u < count ? s.words[i * SUBS + u] : 0u;
    }
#pragma unroll
    for (int k = 0; k < 4 * ROUNDS; ++k) total += s.seg[k];
    __syncthreads();
    return total;
}

// ---------------------------------------------------------------------------------------------------------------------
// Stages: what a work-group's four wavefronts share
// ---------------------------------------------------------------------------------------------------------------------
// SUBS tiles of 32 rows of two tensors (K and V; Q and dO).  fp32 heads of 64 features and more have one tile a stage: their images take
// three times the LDS.
template <class T, int D>
struct CrossStage {
    typedef BiasTile<T, D> TL;
    static constexpr int SUBS = sizeof(T) == 4 && D >= 64 ? 1 : 2, ROWS = 32 * SUBS;
    static constexpr int BYTES = 2 * SUBS * TL::BYTES;  // the first tensor's tiles, then the second's
    static constexpr int N = ROWS * TL::CPR / 256;      // pieces of each tensor a thread moves
    static_assert(N * 256 == ROWS * TL::CPR, "whole pieces");
    PieceInFlight<T> x[N], y[N];
    template <class S>
    __device__ __forceinline__ void load(const S& xs, const S& ys, int first, int tid) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int n = 256 * i + tid, r = n / TL::CPR, c = n % TL::CPR;
            x[i].load(xs.r, xs.at(first, r, 8 * c * (int)sizeof(T)));
            y[i].load(ys.r, ys.at(first, r, 8 * c * (int)sizeof(T)));
        }
    }
    // word[s]: which rows of tile s take part; the others become zeros
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

// bf16 stages go from global memory straight into LDS (tile_kernels.h: loads in assembly blocks, waited for with wait_vm), which takes no
// registers and no LDS stores.  Wavefront w has rows 16 w .. 16 w + 15 of both tensors, 1 KB an instruction; a lane asks for the piece that
// belongs to its place in LDS.  Rows that take no part are overwritten with zeros when they have arrived.
template <int D>
struct CrossStage<__bf16, D> {
    typedef BiasTile<__bf16, D> TL;
    static constexpr int SUBS = 2, ROWS = 64, BYTES = 2 * SUBS * TL::BYTES;
    static constexpr int AT_ONCE = 1024 / TL::ROW, N = 16 / AT_ONCE;  // rows an instruction moves, instructions a tensor
    template <class S>
    __device__ static __forceinline__ void ask(const S& xs, const S& ys, int first, char* buf, int w, int l) {
        const u32x4 xr = cross_words(xs, first), yr = cross_words(ys, first);
        const unsigned at = lds_address(buf) + 16 * w * TL::ROW;
        if constexpr (D == 128) asm volatile("" : "+v"(l));  // (the lane's places made anew: kept, they are registers that the column pass spills)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = 16 * w + AT_ONCE * i + l / TL::CPR, byte = 16 * ((l % TL::CPR) ^ TL::swz(r & 31));
            load(xr, at + 1024 * i, cross_lane(xs, first, r, byte));
            load(yr, at + SUBS * TL::BYTES + 1024 * i, cross_lane(ys, first, r, byte));
        }
    }
    __device__ static __forceinline__ void load(u32x4 r, unsigned lds, int voff) {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(r) : "memory");
    }
    __device__ static __forceinline__ void arrived(char* buf, const unsigned (&word)[SUBS], int w, int l) {
        wait_vm<0>();
        if ((word[0] & word[1]) == ~0u) return;
        const unsigned mine = word[w >> 1] >> (16 * (w & 1));
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = AT_ONCE * i + l / TL::CPR;
            if ((mine >> r) & 1u) continue;
            char* const at = buf + (16 * w + r) * TL::ROW + 16 * (l % TL::CPR);
            *reinterpret_cast<u32x4*>(at) = u32x4{0, 0, 0, 0};
            *reinterpret_cast<u32x4*>(at + SUBS * TL::BYTES) = u32x4{0, 0, 0, 0};
        }
    }
};

template <class T, int D>
constexpr int cross_stages_bytes() {
    const int stages = 2 * CrossStage<T, D>::BYTES, merge = merge_floats<D>() * 4;
    return stages > merge ? stages : merge;
}

struct NothingElseToFetch {
    __device__ __forceinline__ void load(int) {}
    __device__ __forceinline__ void store(int) {}
};

// The stages of a piece of the other side, one after the other, in two buffers taken in turn (one barrier a stage; of bf16 stages the buffer is
// known at compile time, so that the operands' LDS addresses are constants beside the lane's, and fp32 bodies are too large to stand
// there twice).  body(words, buffer, which).
template <class T, int D, bool KEYS, class S, class Fetched, class Body>
__device__ __forceinline__ void cross_walk(const CrossCall& a, CrossLds& sc, const CrossItem& it, const S& xs, const S& ys, char* lds, int tid,
                                           Fetched&& fetched, Body&& body) {
    typedef CrossStage<T, D> ST;
    constexpr bool DIRECT = sizeof(T) == 2;
    const bool listed = KEYS && a.mask;
    const int rows = KEYS ? a.Lk : a.rows, w = uniform(tid >> 6), l = tid & 63;
    const int from = it.split * a.per_split, to = min((rows + 31) / 32, from + a.per_split), chunk = listed ? CHUNK : a.per_split;
    for (int first = from; first < to; first += chunk) {
        const int count = min(chunk, to - first);
        const int n = listed ? cross_scan<ST::SUBS>(a, sc, it.b, first, count, tid) : (count + ST::SUBS - 1) / ST::SUBS;
        ST st;
        // A stage's place and words are read from the list while the one two before it is worked on: read where they are needed, they cost a padded
        // call a tenth of its time (128 heads of 1024 x 2048, three quarters of the keys: forward 90 us, so 82).
        struct Entry {
            int unit;
            unsigned word[ST::SUBS];
        };
        auto look_up = [&](int i) __attribute__((always_inline)) {
            Entry e;
            e.unit = i;
            if (listed) {
                const int at = min(i, n - 1);
                e.unit = sc.list[at];
#pragma unroll
                for (int u = 0; u < ST::SUBS; ++u) e.word[u] = sc.of[at * ST::SUBS + u];
            }
            return e;
        };
        Entry now, next;
        auto ask = [&](char* buf) __attribute__((always_inline)) {  // the stage of `now`
            now.unit = uniform(now.unit);
            const int row = (first + now.unit * ST::SUBS) * 32;
#pragma unroll
            for (int u = 0; u < ST::SUBS; ++u)
                now.word[u] = listed ? (unsigned)uniform((int)now.word[u]) : now.unit * ST::SUBS + u < count ? tail_word(rows - row - 32 * u) : 0u;
            if constexpr (DIRECT) ST::ask(xs, ys, row, buf, w, l);
            else st.load(xs, ys, row, tid);
            fetched.load(row);
        };
        auto step = [&](int i, auto which) __attribute__((always_inline)) {
            const int P = which;
            unsigned word[ST::SUBS];
#pragma unroll
            for (int u = 0; u < ST::SUBS; ++u) word[u] = now.word[u];
            char* const buf = lds + P * ST::BYTES;
            if constexpr (DIRECT) ST::arrived(buf, word, w, l);
            else st.store(buf, word, tid);
            fetched.store(P);
            group_barrier();
            if (i + 1 < n) {
                now = next;
                ask(lds + (1 - P) * ST::BYTES);
                next = look_up(i + 2);
            }
            body(word, buf, which);
        };
        if (n > 0) {
            now = look_up(0);
            next = look_up(1);
            ask(lds);
        }
        if constexpr (DIRECT) {
            for (int i = 0; i < n; i += 2) {
                step(i, std::integral_constant<int, 0>());
                if (i + 1 < n) step(i + 1, std::integral_constant<int, 1>());
            }
        } else {
            for (int i = 0; i < n; ++i) step(i, i & 1);
        }
    }
}

// A wavefront's 32 x D result acc[c][r] (lane (li, h): row li, feature 32 c + acc_row(r, h)), scaled by the lane's f, through its part of
// red; out(row, eighth, values).
template <int D, class Out>
__device__ __forceinline__ void cross_store(const f32x16 (&acc)[D / 32], float f, float* red, int w, int l, Out&& out) {
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
// eighth j of a row of a tensor
template <class T, int D>
__device__ __forceinline__ void cross_put(const char* row, int j, const float (&x)[D / 8]) {
    store_values<T, D / 8>(const_cast<char*>(row) + j * (D / 8) * sizeof(T), x);
}
template <int D>
__device__ __forceinline__ void cross_leave(float* slot, int row, int j, const float (&x)[D / 8]) {
    store_values<float, D / 8>(reinterpret_cast<char*>(slot + row * D + j * (D / 8)), x);
}

// -------------------------------------------------------------------------------------------------
// Forward
// -------------------------------------------------------------------------------------------------
// The softmax of one wavefront's rows, a lane each (twice: half-wave h has the keys of its accumulator rows).
template <class T, int D>
struct CrossSoftmax {
    typedef BiasTile<T, D> TL;
    f32x16 o[D / 32];
    float m = -__builtin_inff(), z = 0.f;
    __device__ __forceinline__ CrossSoftmax() {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) o[c] = splat16(0.f);
    }
    // the maximum of N tiles' products s, keys that are left out at -infinity
    template <int N>
    __device__ __forceinline__ void raise(f32x16 (&s)[N], const unsigned (&word)[N], float c2, int h) {
        float mt = -__builtin_inff();
#pragma unroll
        for (int u = 0; u < N; ++u) {
            if (word[u] != ~0u) {
                const unsigned mine = word[u] >> (4 * h);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[u][r] = (mine >> (8 * (r >> 2) + (r & 3))) & 1u ? s[u][r] : -__builtin_inff();
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) mt = fmaxf(mt, s[u][r]);
        }
        mt = half_swap_max(mt) * c2;
        if (__any(mt > m + CROSS_LAZY)) {
            const float up = fmaxf(m, mt);
            const float f = up == m ? 1.f : __builtin_amdgcn_exp2f(m - up);  // equal: also -infinity twice
            m = up;
            z *= f;
#pragma unroll
            for (int c = 0; c < D / 32; ++c)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[c][r] *= f;
        }
    }
    __device__ __forceinline__ float base() const { return m == -__builtin_inff() ? 0.f : m; }
    __device__ __forceinline__ void weights(const f32x16& s, float c2, float minus, float (&p)[16]) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            p[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c2, minus));
            z += p[r];
        }
    }
};

// Wavefronts a SIMD that the registers are for.
template <class T, int D>
constexpr int cross_forward_waves() { return D == 128 ? (sizeof(T) == 2 ? 2 : 1) : sizeof(T) == 2 ? 3 : 2; }
// (Row pass, D = 128, bf16, whose operands are read as the products need them: 256 heads of 2048 x 4096 2050 us with one wavefront, 1555 with two.
// Three at D = 64: 900 and 815.)
template <class T, int D>
constexpr int cross_row_waves() { return sizeof(T) == 2 ? (D == 128 ? 2 : 3) : D == 32 ? 2 : 1; }
template <class T, int D>
constexpr int cross_backward_waves() { return sizeof(T) == 2 ? (D == 128 ? 1 : 2) : D == 32 ? 2 : 1; }

// 128 rows to a work-group, 32 to each of its wavefronts.
template <class T, int D>
__global__ __launch_bounds__(256, (cross_forward_waves<T, D>())) void cross_forward_kernel(CrossCall a) {
    typedef BiasTile<T, D> TL;
    typedef CrossStage<T, D> ST;
    constexpr int SUBS = ST::SUBS;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    CrossLds& sc = *reinterpret_cast<CrossLds*>(lds + cross_stages_bytes<T, D>());
    const int tid = threadIdx.x, w = uniform(tid >> 6), l = tid & 63, li = l & 31, h = l >> 5;
    const CrossItem it(a, gridDim.x);
    const int q0 = it.strip * 128 + 32 * w;
    const bool some = q0 < a.rows;
    const typename TL::Row q = TL::load(a.row(a.q, it.b, it.g, min(q0 + li, a.rows - 1)), h, q0 + li < a.rows);
    const typename TL::At at = TL::at(l);
    const float c2 = a.scale * LOG2E;
    q.settled();
    CrossSoftmax<T, D> x;
    typedef CrossSource<T, D, true> S;
    cross_walk<T, D, true>(a, sc, it, S(a, a.k, it.b, it.g), S(a, a.v, it.b, it.g), lds, tid, NothingElseToFetch(),
        [&](const unsigned (&word)[SUBS], const char* buf, auto) __attribute__((always_inline)) {
            if (!some) return;
            f32x16 s[SUBS];
            typename TL::Row kr[SUBS];
#pragma unroll
            for (int u = 0; u < SUBS; ++u) kr[u] = TL::rows(buf + u * TL::BYTES, at);
            issue_order();
#pragma unroll
            for (int u = 0; u < SUBS; ++u) s[u] = TL::feat(kr[u], q);
            x.raise(s, word, c2, h);
            const float minus = -x.base();
#pragma unroll
            for (int u = 0; u < SUBS; ++u) {
                float p[16];
                x.weights(s[u], c2, minus, p);
                TL::add_t(TL::columns(buf + (SUBS + u) * TL::BYTES, at), p, x.o);
            }
        });
    const float z = half_swap_sum(x.z);
    __syncthreads();  // the stages are done with
    if (!some) return;
    if (a.splits > 1) {
        float* slot = a.part + it.slot(a, a.rows, q0) * cross_slot<D>();
        if (h == 0) {
            slot[32 * D + li] = x.m;
            slot[32 * D + 32 + li] = z;
        }
        cross_store<D>(x.o, 1.f, reinterpret_cast<float*>(lds), w, l, [&](int row, int j, float (&v)[D / 8]) {
            if (q0 + row < a.rows) cross_leave<D>(slot, row, j, v);
        });
        return;
    }
    if (h == 0 && q0 + li < a.rows)
        a.lse[(size_t)it.bg * a.rows + q0 + li] = z == 0.f ? __builtin_inff() : x.m + __builtin_amdgcn_logf(z);
    cross_store<D>(x.o, z == 0.f ? 0.f : 1.f / z, reinterpret_cast<float*>(lds), w, l, [&](int row, int j, float (&v)[D / 8]) {
        if (q0 + row < a.rows) cross_put<T, D>(a.row(a.o, it.b, it.g, q0 + row), j, v);
    });
}

// what rounding to bf16 takes from p
__device__ __forceinline__ void cross_rest(float (&p)[16]) {
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
        const unsigned hi = pack_bf16(p[r], p[r + 1]);
        p[r] -= bf16_lo(hi);
        p[r + 1] -= bf16_hi(hi);
    }
}
// out += X^T . W of bf16 tiles with W as the sum of two bf16 numbers (fp32 tiles have three images, and no second product here).  bf16 calls of a token
// wait for memory, so that the second product and its 40 vector instructions cost nothing there (2048 keys 8.6 us with either); it goes with every
// strip of 32, and the rounding of the weights is gone from their results: errors of 0.0017, that of the result's own rounding, against 0.0024.
template <class TL, class Columns, int N>
__device__ __forceinline__ void cross_add_fine(const Columns& xt, const float (&p)[16], f32x16 (&out)[N]) {
    TL::add_t(xt, p, out);
    if constexpr (TL::IM == 1) {
        float rest[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) rest[r] = p[r];
        cross_rest(rest);
        TL::add_t(xt, rest, out);
    }
}

// Few rows: 32 of them to a work-group, and its wavefronts take every fourth tile of the keys, each through its own part of LDS, so that
// nothing waits for a barrier inside the walk.
template <class T, int D>
constexpr int cross_own_tiles() { return sizeof(T) == 4 && D == 128 ? 1 : 2; }  // (two fp32 tiles of 128 features for four wavefronts do not fit a CU)
template <class T, int D>
constexpr int cross_tiles_bytes() {
    const int tiles = 4 * cross_own_tiles<T, D>() * BiasTile<T, D>::BYTES, merge = merge_floats<D>() * 4;
    return tiles > merge ? tiles : merge;
}
// Wavefront w of piece s has tiles 4 s + w, 4 (s + splits) + w, ...: what padding leaves is dealt evenly (in ranges of tiles, a piece could have
// none).  It makes the words of its tiles itself, from mask values that were asked for two tiles ahead; K and V are one tile ahead.
// body(tile's first key, word, put_k, put_v): for all tiles, those without a key (a word of 0) among them if EVERY; put_k(), once for tiles with a
// key, brings K and V to LDS and asks for the next; with one tile it brings K, and put_v(), which comes first or not (V_FIRST), V.
template <class T, int D, bool EVERY, bool V_FIRST, class Body>
__device__ __forceinline__ void cross_few_walk(const CrossCall& a, const CrossItem& it, char* tk, char* tv, int w, int l, Body&& body) {
    const HeadBuf kh = HeadBuf::of<T, D>(a.k, it.b, it.g, a.Lk), vh = HeadBuf::of<T, D>(a.v, it.b, it.g, a.Lk);
    const int tiles = (a.Lk + 31) / 32, step = 4 * a.splits;
    const size_t row = (size_t)it.b * a.Lk;
    auto ask = [&](int tile) __attribute__((always_inline)) -> unsigned {  // (a float of 0 or -0 and a byte of 0 are left out)
        const int key = tile * 32 + (l & 31);
        if (!a.mask || key >= a.Lk) return 0u;
        return a.mask_bytes == 4 ? reinterpret_cast<const unsigned*>(a.mask)[row + key] << 1 : reinterpret_cast<const unsigned char*>(a.mask)[row + key];
    };
    auto word_of = [&](int tile, unsigned asked) __attribute__((always_inline)) -> unsigned {
        if (tile >= tiles) return 0u;
        return a.mask ? (unsigned)__ballot(asked != 0) : tail_word(a.Lk - tile * 32);
    };
    // With one tile (ONE) the tensors take turns: what is put second is asked for when the first one has been put, so that one of them is in flight.
    constexpr bool ONE = cross_own_tiles<T, D>() == 1;
    TileInFlight<T, D> fk, other;
    TileInFlight<T, D>& fv = ONE ? fk : other;
    auto fetch = [&](int tile) __attribute__((always_inline)) {
        if (!ONE || !V_FIRST) fk.load(kh, tile * 32, l);
        if (!ONE || V_FIRST) fv.load(vh, tile * 32, l);
    };
    int tile = 4 * it.split + w;
    unsigned asked = ask(tile), next = ask(tile + step), word = word_of(tile, asked);
    if (word) fetch(tile);
    for (; tile < tiles; tile += step) {
        const unsigned now = word;
        word = word_of(tile + step, next);
        next = ask(tile + 2 * step);
        auto put_k = [&]() __attribute__((always_inline)) {
            wave_lds_order();
            fk.store(tk, now, l);
            if (!ONE) fv.store(tv, now, l);
            wave_lds_order();
            if (ONE && !V_FIRST) fv.load(vh, tile * 32, l);
            else if (word && ONE) fv.load(vh, (tile + step) * 32, l);
            else if (word) fetch(tile + step);
        };
        auto put_v = [&]() __attribute__((always_inline)) {  // (ONE)
            wave_lds_order();
            fv.store(tv, now, l);
            wave_lds_order();
            if (V_FIRST) fk.load(kh, tile * 32, l);
            else if (word) fk.load(kh, (tile + step) * 32, l);
        };
        if (!now && word) fetch(tile + step);
        if (EVERY || now) body(tile * 32, now, put_k, put_v);
    }
}

template <class T, int D>
__global__ __launch_bounds__(256, (cross_backward_waves<T, D>())) void cross_forward_few_kernel(CrossCall a) {
    typedef BiasTile<T, D> TL;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ float ml[4][2][32], inv[32];
    const int tid = threadIdx.x, w = uniform(tid >> 6), l = tid & 63, li = l & 31, h = l >> 5;
    const CrossItem it(a, gridDim.x);
    const int q0 = it.strip * 32;
    const typename TL::Row q = TL::load(a.row(a.q, it.b, it.g, min(q0 + li, a.rows - 1)), h, q0 + li < a.rows);
    const typename TL::At at = TL::at(l);
    constexpr int TILES = cross_own_tiles<T, D>();
    char* tk = lds + w * TILES * TL::BYTES;
    char* tv = tk + (TILES - 1) * TL::BYTES;
    const float c2 = a.scale * LOG2E;
    q.settled();
    CrossSoftmax<T, D> x;
    cross_few_walk<T, D, false, false>(a, it, tk, tv, w, l, [&](int, unsigned word, auto&& put_k, auto&& put_v) __attribute__((always_inline)) {
        put_k();
        const typename TL::Row kr = TL::rows(tk, at);
        typename TL::Columns vt;
        if (TL::EARLY) vt = TL::columns(tv, at);
        issue_order();
        f32x16 s[1] = {TL::feat(kr, q)};
        const unsigned words[1] = {word};
        x.raise(s, words, c2, h);
        float p[16];
        x.weights(s[0], c2, -x.base(), p);
        if (TILES == 1) put_v();
        if (!TL::EARLY) vt = TL::columns(tv, at);
        cross_add_fine<TL>(vt, p, x.o);
    });
    // the four wavefronts' parts
    const float z = half_swap_sum(x.z);
    if (h == 0) {
        ml[w][0][li] = x.m;
        ml[w][1][li] = z;
    }
    __syncthreads();
    float M = ml[0][0][li];
#pragma unroll
    for (int k = 1; k < 4; ++k) M = fmaxf(M, ml[k][0][li]);
    const float base = M == -__builtin_inff() ? 0.f : M;
    float Z = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) Z += ml[k][1][li] * __builtin_amdgcn_exp2f(ml[k][0][li] - base);
    const float f = __builtin_amdgcn_exp2f(x.m - base);
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) x.o[c][r] *= f;
    float v[D / 8];
    merge_waves<D>(x.o, reinterpret_cast<float*>(lds), tid, v);
    const int row = tid >> 3, j = tid & 7;
    if (a.splits > 1) {
        float* slot = a.part + it.slot(a, a.rows, q0) * cross_slot<D>();
        if (q0 + row < a.rows) cross_leave<D>(slot, row, j, v);
        if (w == 0 && h == 0) {
            slot[32 * D + li] = M;
            slot[32 * D + 32 + li] = Z;
        }
        return;
    }
    if (w == 0 && h == 0) {
        inv[li] = Z == 0.f ? 0.f : 1.f / Z;
        if (q0 + li < a.rows) a.lse[(size_t)it.bg * a.rows + q0 + li] = Z == 0.f ? __builtin_inff() : M + __builtin_amdgcn_logf(Z);
    }
    __syncthreads();
    if (q0 + row < a.rows) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) v[i] *= inv[row];
        cross_put<T, D>(a.row(a.o, it.b, it.g, q0 + row), j, v);
    }
}

// The pieces of a row, added up in a fixed order; a lane has four features.  MANY (more than eight pieces): a work-group has one row, and its
// groups of D / 4 lanes every GROUPS-th piece.  Else a group has a row of its own and all of its pieces.  (16 rows in 64 pieces, d = 128: 4.5 us,
// and 18 with all pieces to a lane; 32768 rows in two pieces, d = 64: a wavefront a row 17.)
template <int D, bool MANY>
struct CrossJoin {
    static constexpr int COLS = D / 4, SETS = 256 / COLS, GROUPS = MANY ? SETS : 1, ROWS = MANY ? 1 : SETS;
    int row, col, group;  // of the work-group's ROWS, four features, which of the GROUPS
    __device__ __forceinline__ CrossJoin(int tid) : row(MANY ? 0 : tid / COLS), col(tid % COLS), group(MANY ? tid / COLS : 0) {}
    // sum over the pieces of f(piece) * the row of slot `piece`; whole in the lanes of group 0
    template <class F>
    __device__ __forceinline__ f32x4 sum(const float* rows, int pieces, int stride, f32x4* red, F&& f) const {
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
        for (int k = group; k < pieces; k += GROUPS) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(rows + (size_t)k * stride + 4 * col);
            const float by = f(k);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = fmaf(v[e], by, x[e]);
        }
        if constexpr (MANY) {
            red[group * COLS + col] = x;
            __syncthreads();
            if (group == 0)
#pragma unroll
                for (int g = 1; g < GROUPS; ++g)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] += red[g * COLS + col][e];
        }
        return x;
    }
};
// four values to memory, rounded once
template <class T>
__device__ __forceinline__ void cross_put4(const char* row, int col, f32x4 x) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<f32x4*>(const_cast<char*>(row))[col] = x;
    } else {
        bf16x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (__bf16)x[e];
        reinterpret_cast<bf16x4*>(const_cast<char*>(row))[col] = v;
    }
}

template <class T, int D, bool MANY>
__global__ __launch_bounds__(256) void cross_merge_kernel(CrossCall a) {
    typedef CrossJoin<D, MANY> J;
    __shared__ f32x4 red[MANY ? 256 : 1];
    __shared__ float by[MANY ? 64 : 1];
    const int tid = threadIdx.x, l = tid & 63;
    const J j(tid);
    const int sets = (a.rows + J::ROWS - 1) / J::ROWS, bg = blockIdx.x / sets, r = min((int)(blockIdx.x - bg * sets) * J::ROWS + j.row, a.rows - 1);
    const float* slot = a.part + ((size_t)bg * ((a.rows + 31) / 32) + r / 32) * a.splits * cross_slot<D>();
    const float* stats = slot + 32 * D + r % 32;  // of the first piece
    float M = -__builtin_inff(), Z = 0.f;
    f32x4 x;
    if constexpr (MANY) {  // a piece a lane (there are no more than 64)
        const bool have = l < a.splits;
        const float* mine = stats + (size_t)min(l, a.splits - 1) * cross_slot<D>();
        const float m = have ? mine[0] : -__builtin_inff(), z = have ? mine[32] : 0.f;
        M = m;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
        const float f = __builtin_amdgcn_exp2f(m - (M == -__builtin_inff() ? 0.f : M));
        Z = z * f;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) Z += __shfl_xor(Z, o, 64);
        if (tid < 64) by[l] = f;
        __syncthreads();
        x = j.sum(slot + (r % 32) * D, a.splits, cross_slot<D>(), red, [&](int k) { return by[k]; });
    } else {
        float m[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            m[k] = k < a.splits ? stats[(size_t)k * cross_slot<D>()] : -__builtin_inff();
            M = fmaxf(M, m[k]);
        }
        const float base = M == -__builtin_inff() ? 0.f : M;
        x = j.sum(slot + (r % 32) * D, a.splits, cross_slot<D>(), red, [&](int k) {
            const float f = __builtin_amdgcn_exp2f(stats[(size_t)k * cross_slot<D>()] - base);
            Z = fmaf(stats[(size_t)k * cross_slot<D>() + 32], f, Z);
            return f;
        });
    }
    if (j.group != 0) return;
    const float inv = Z == 0.f ? 0.f : 1.f / Z;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] *= inv;
    cross_put4<T>(a.row(a.o, bg / a.G, bg % a.G, r), j.col, x);
    if (j.col == 0) a.lse[(size_t)bg * a.rows + r] = Z == 0.f ? __builtin_inff() : M + __builtin_amdgcn_logf(Z);
}

// -------------------------------------------------------------------------------------------------
// Backward, rows: dQ and D
// -------------------------------------------------------------------------------------------------
// dS of a tile: rows keys, lanes queries.  minus_lse of the lane's row; dp: dP - D.
__device__ __forceinline__ void cross_ds(const f32x16& s, const f32x16& dp, float c2, float minus_lse, unsigned word, int h, float (&ds)[16]) {
#pragma unroll
    for (int r = 0; r < 16; ++r) ds[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c2, minus_lse)) * dp[r];
    if (word != ~0u) {
        const unsigned mine = word >> (4 * h);
#pragma unroll
        for (int r = 0; r < 16; ++r) ds[r] = (mine >> (8 * (r >> 2) + (r & 3))) & 1u ? ds[r] : 0.f;
    }
}

// FINE (bf16): dS in two bf16 numbers (cross_add_fine).  D = dO . O, of an O that is rounded, is the further off against dP - D the fewer keys there are,
// and with dS rounded too the gradients of a call of few keys are half as far off again as their own rounding (100 keys, d = 64: 0.0026 and
// 0.0017; so 0.0020).
template <class T, int D, bool FINE>
__global__ __launch_bounds__(256, (cross_row_waves<T, D>())) void cross_backward_row_kernel(CrossCall a) {
    typedef BiasTile<T, D> TL;
    typedef CrossStage<T, D> ST;
    constexpr int SUBS = ST::SUBS;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    CrossLds& sc = *reinterpret_cast<CrossLds*>(lds + cross_stages_bytes<T, D>());
    const int tid = threadIdx.x, w = uniform(tid >> 6), l = tid & 63, li = l & 31, h = l >> 5;
    const CrossItem it(a, gridDim.x);
    const int q0 = it.strip * 128 + 32 * w, qi = min(q0 + li, a.rows - 1);
    const bool some = q0 < a.rows, there = q0 + li < a.rows;
    const typename TL::Row q = TL::load(a.row(a.q, it.b, it.g, qi), h, there);
    const typename TL::Row go = TL::load(a.row(a.dout, it.b, it.g, qi), h, there);
    const size_t stat = (size_t)it.bg * a.rows + qi;
    const float minus_lse = there ? -a.lse[stat] : -__builtin_inff();
    const float delta = half_swap_sum(TL::dot(go, TL::load(a.row(a.o, it.b, it.g, qi), h, there)));
    if (it.split == 0 && h == 0 && there) a.delta[stat] = delta;
    const typename TL::At at = TL::at(l);
    const float c2 = a.scale * LOG2E;
    const f32x16 minus = splat16(-delta);
    q.settled();
    go.settled();
    f32x16 dq[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) dq[c] = splat16(0.f);
    typedef CrossSource<T, D, true> S;
    cross_walk<T, D, true>(a, sc, it, S(a, a.k, it.b, it.g), S(a, a.v, it.b, it.g), lds, tid, NothingElseToFetch(),
        [&](const unsigned (&word)[SUBS], const char* buf, auto) __attribute__((always_inline)) {
            if (!some) return;
#pragma unroll
            for (int u = 0; u < SUBS; ++u) {
                if (word[u] == 0) continue;
                const char *tk = buf + u * TL::BYTES, *tv = buf + (SUBS + u) * TL::BYTES;
                const typename TL::Row kr = TL::rows(tk, at), vr = TL::rows(tv, at);
                typename TL::Columns kt;
                if (D < 128) issue_order();
                const f32x16 s = TL::feat(kr, q);
                if (D == 128) issue_order();
                const f32x16 dp = TL::feat(vr, go, D == 128 ? splat16(-delta) : minus);
                if (D == 128) issue_order();
                if (TL::EARLY && D < 128) {
                    kt = TL::columns(tk, at);
                    read_behind_products<D / 8, D / 8>();
                }
                float ds[16];
                cross_ds(s, dp, c2, minus_lse, word[u], h, ds);
                if (!TL::EARLY || D == 128) kt = TL::columns(tk, at);
                if constexpr (FINE) cross_add_fine<TL>(kt, ds, dq);
                else TL::add_t(kt, ds, dq);
            }
        });
    __syncthreads();  // the stages are done with
    if (!some) return;
    float* slot = a.part + it.slot(a, a.rows, q0) * (32 * D);
    cross_store<D>(dq, a.scale, reinterpret_cast<float*>(lds), w, l, [&](int row, int j, float (&v)[D / 8]) {
        if (q0 + row >= a.rows) return;
        if (a.splits > 1) cross_leave<D>(slot, row, j, v);
        else cross_put<T, D>(a.row(a.dq, it.b, it.g, q0 + row), j, v);
    });
}

// A wavefront's tile of rows of Q or dO on its way to LDS (TileInFlight, which has the rows of one head).
template <class T, int D>
struct RowsInFlight {
    typedef BiasTile<T, D> TL;
    PieceInFlight<T> x[TL::CPR / 2];
    template <class S>
    __device__ __forceinline__ void load(const S& from, int first, int l) {
#pragma unroll
        for (int i = 0; i < TL::CPR / 2; ++i) x[i].load(from.r, from.at(first, (64 * i + l) / TL::CPR, 8 * (l % TL::CPR) * (int)sizeof(T)));
    }
    __device__ __forceinline__ void store(char* tile, unsigned word, int l) const {
#pragma unroll
        for (int i = 0; i < TL::CPR / 2; ++i) x[i].template store<D, false>(tile, (64 * i + l) / TL::CPR, l % TL::CPR, (word >> ((64 * i + l) / TL::CPR)) & 1u);
    }
};

// Where the operands of 32 rows of their own are too many registers (fp32, 128 features: 192), a work-group's wavefronts read them from two tiles that
// they share.
template <class T, int D>
constexpr int cross_shared_bytes() { return cross_own_tiles<T, D>() == 1 ? 2 * BiasTile<T, D>::BYTES : 0; }
template <class T, int D, class S>
__device__ __forceinline__ void cross_share(char* tiles, const S& xs, const S& ys, int first, int rows, int w, int l) {
    if (w < 2) {
        RowsInFlight<T, D> x;
        x.load(w ? ys : xs, first, l);
        x.store(tiles + w * BiasTile<T, D>::BYTES, tail_word(rows - first), l);
    }
    __syncthreads();
}

// Strips of 32 rows, as in cross_forward_few_kernel.
template <class T, int D>
__global__ __launch_bounds__(256, (cross_backward_waves<T, D>())) void cross_backward_row_few_kernel(CrossCall a) {
    typedef BiasTile<T, D> TL;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, w = uniform(tid >> 6), l = tid & 63, li = l & 31, h = l >> 5;
    const CrossItem it(a, gridDim.x);
    const int q0 = it.strip * 32, qi = min(q0 + li, a.rows - 1);
    const bool there = q0 + li < a.rows;
    constexpr int TILES = cross_own_tiles<T, D>();
    char* const shared = lds + cross_tiles_bytes<T, D>();
    typename TL::Row q, go = TL::load(a.row(a.dout, it.b, it.g, qi), h, there);
    const size_t stat = (size_t)it.bg * a.rows + qi;
    const float minus_lse = there ? -a.lse[stat] : -__builtin_inff();
    const float delta = half_swap_sum(TL::dot(go, TL::load(a.row(a.o, it.b, it.g, qi), h, there)));
    if (it.split == 0 && tid < 32 && there) a.delta[stat] = delta;
    const typename TL::At at = TL::at(l);
    char* tk = lds + w * TILES * TL::BYTES;
    char* tv = tk + (TILES - 1) * TL::BYTES;
    const float c2 = a.scale * LOG2E;
    const f32x16 minus = splat16(-delta);
    if constexpr (TILES == 1) {
        typedef CrossSource<T, D, false> S;
        cross_share<T, D>(shared, S(a, a.q, it.b, it.g), S(a, a.dout, it.b, it.g), q0, a.rows, w, l);
    } else {
        q = TL::load(a.row(a.q, it.b, it.g, qi), h, there);
        q.settled();
        go.settled();
    }
    f32x16 dq[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) dq[c] = splat16(0.f);
    cross_few_walk<T, D, false, true>(a, it, tk, tv, w, l, [&](int, unsigned word, auto&& put_k, auto&& put_v) __attribute__((always_inline)) {
        f32x16 s, dp;
        typename TL::Columns kt;
        if constexpr (TILES == 1) {
            int same = 0;  // (not so to the compiler, which would keep what the shared tiles hold in registers)
            asm volatile("" : "+v"(same));
            put_v();
            dp = TL::feat(TL::rows(tv, at), TL::rows(shared + TL::BYTES + same, at), minus);
            put_k();
            s = TL::feat(TL::rows(tk, at), TL::rows(shared + same, at));
        } else {
            put_k();
            const typename TL::Row kr = TL::rows(tk, at), vr = TL::rows(tv, at);
            if (TL::EARLY) kt = TL::columns(tk, at);
            issue_order();
            s = TL::feat(kr, q);
            dp = TL::feat(vr, go, minus);
        }
        float ds[16];
        cross_ds(s, dp, c2, minus_lse, word, h, ds);
        if (!TL::EARLY) kt = TL::columns(tk, at);
        cross_add_fine<TL>(kt, ds, dq);
    });
    __syncthreads();  // the tiles are done with
    float v[D / 8];
    merge_waves<D>(dq, reinterpret_cast<float*>(lds), tid, v);
    const int row = tid >> 3, j = tid & 7;
    if (q0 + row >= a.rows) return;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) v[i] *= a.scale;
    if (a.splits > 1) cross_leave<D>(a.part + it.slot(a, a.rows, q0) * (32 * D), row, j, v);
    else cross_put<T, D>(a.row(a.dq, it.b, it.g, q0 + row), j, v);
}

template <class T, int D, bool MANY>
__global__ __launch_bounds__(256) void cross_merge_row_kernel(CrossCall a) {
    typedef CrossJoin<D, MANY> J;
    __shared__ f32x4 red[MANY ? 256 : 1];
    const int tid = threadIdx.x;
    const J j(tid);
    const int sets = (a.rows + J::ROWS - 1) / J::ROWS, bg = blockIdx.x / sets, r = min((int)(blockIdx.x - bg * sets) * J::ROWS + j.row, a.rows - 1);
    const float* slot = a.part + ((size_t)bg * ((a.rows + 31) / 32) + r / 32) * a.splits * (32 * D);
    const f32x4 x = j.sum(slot + (r % 32) * D, a.splits, 32 * D, red, [](int) { return 1.f; });
    if (j.group == 0) cross_put4<T>(a.row(a.dq, bg / a.G, bg % a.G, r), j.col, x);
}

// -------------------------------------------------------------------------------------------------
// Backward of few rows, in one pass over the keys
// -------------------------------------------------------------------------------------------------
// All rows of a group in one strip of 32: a tile's dK and dV are then whole after its own products, and K and V are read once for
// all three gradients (the two passes read them twice: 64 fp32 heads of 4096 padded keys, 16 rows, d = 32: the training step 82 us then, and 66).  dQ wants the
// rows as lanes and dK, dV the keys, so both products over the head dimension are formed twice, with their operands exchanged: they
// lie in registers either way.  Every wavefront takes every fourth tile, leaves its dK and dV and keeps dQ.  Bound by a tile's work, seven products of 32 rows
// however many there are, rather than by memory: those heads take 34 us, 3.4 TB/s, and in bf16 20 us for half of the bytes.
template <class T, int D>
constexpr int cross_few_region() {  // a wavefront's tiles of K and V, then its results on their way out
    const int tiles = cross_own_tiles<T, D>() * BiasTile<T, D>::BYTES, out = 32 * (D + 4) * 4;
    return tiles > out ? tiles : out;
}
template <class T, int D>
constexpr int cross_few_bytes() { return 4 * cross_few_region<T, D>() + 2 * BiasTile<T, D>::BYTES + 64 * 4; }

template <class T, int D>
__global__ __launch_bounds__(256, (cross_backward_waves<T, D>())) void cross_backward_few_kernel(CrossCall a) {
    typedef BiasTile<T, D> TL;
    constexpr int TILES = cross_own_tiles<T, D>();
    extern __shared__ __attribute__((aligned(16))) char lds[];
    char* const tq = lds + 4 * cross_few_region<T, D>();
    char* const tg = tq + TL::BYTES;
    float* const stats = reinterpret_cast<float*>(tg + TL::BYTES);
    const int tid = threadIdx.x, w = uniform(tid >> 6), l = tid & 63, li = l & 31, h = l >> 5;
    const CrossItem it(a, gridDim.x);
    const int qi = min(li, a.rows - 1);
    const bool there = li < a.rows;
    if (w < 2) {  // the tiles of Q and dO, for the products over the rows
        typedef CrossSource<T, D, false> S;
        const S from(a, w ? a.dout : a.q, it.b, it.g);
        RowsInFlight<T, D> x;
        x.load(from, 0, l);
        x.store(w ? tg : tq, tail_word(a.rows), l);
    }
    const float minus_lse = there ? -a.lse[(size_t)it.bg * a.rows + qi] : -__builtin_inff();
    const float delta = half_swap_sum(TL::dot(TL::load(a.row(a.dout, it.b, it.g, qi), h, there), TL::load(a.row(a.o, it.b, it.g, qi), h, there)));
    if (tid < 32) {
        stats[li] = minus_lse;
        stats[32 + li] = -delta;
    }
    const typename TL::At at = TL::at(l);
    char* const tk = lds + w * cross_few_region<T, D>();
    char* const tv = tk + (TILES - 1) * TL::BYTES;
    const float c2 = a.scale * LOG2E;
    f32x16 dq[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) dq[c] = splat16(0.f);
    const char *const ok = a.dk.head(it.b, it.g), *const ov = a.dv.head(it.b, it.g);
    __syncthreads();  // the tiles of Q and dO, and the rows' numbers
    cross_few_walk<T, D, true, true>(a, it, tk, tv, w, l, [&](int k0, unsigned word, auto&& put_k, auto&& put_v) __attribute__((always_inline)) {
        float p[16], ds[16];
        // (an offset that is not the same in every turn to the compiler, which would keep what the tiles of Q and dO hold in registers)
        int same = 0;
        asm volatile("" : "+v"(same));
        const float* const st = stats + same + 4 * h;
        if (word) {
            // rows of K and V by the queries, for dQ, and the other way round, for dK and dV
            f32x16 s, dp;
            auto minus_d = [&]() __attribute__((always_inline)) {
                f32x16 x;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 d = *reinterpret_cast<const f32x4*>(st + 32 + 8 * g);
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[4 * g + j] = d[j];
                }
                return x;
            };
            if constexpr (TILES == 1) {
                put_v();
                const f32x16 dp_t = TL::feat(TL::rows(tv, at), TL::rows(tg + same, at), splat16(-delta));
                dp = TL::feat(TL::rows(tg + same, at), TL::rows(tv, at), minus_d());
                put_k();
                cross_ds(TL::feat(TL::rows(tk, at), TL::rows(tq + same, at)), dp_t, c2, minus_lse, word, h, ds);
                cross_add_fine<TL>(TL::columns(tk, at), ds, dq);
                issue_order();
                s = TL::feat(TL::rows(tq + same, at), TL::rows(tk, at));
            } else {
                put_k();
                cross_ds(TL::feat(TL::rows(tk, at), TL::rows(tq + same, at)), TL::feat(TL::rows(tv, at), TL::rows(tg + same, at), splat16(-delta)), c2,
                         minus_lse, word, h, ds);
                cross_add_fine<TL>(TL::columns(tk, at), ds, dq);
                issue_order();
                s = TL::feat(TL::rows(tq + same, at), TL::rows(tk, at));
                dp = TL::feat(TL::rows(tg + same, at), TL::rows(tv, at), minus_d());
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 e = *reinterpret_cast<const f32x4*>(st + 8 * g);
#pragma unroll
                for (int j = 0; j < 4; ++j) p[4 * g + j] = __builtin_amdgcn_exp2f(fmaf(s[4 * g + j], c2, e[j]));
            }
            // a key that is left out was stored as zeros, and its P is exp2(-lse)
            const bool key = (word >> li) & 1u;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                ds[r] = key ? p[r] * dp[r] : 0.f;
                p[r] = key ? p[r] : 0.f;
            }
        } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) p[r] = ds[r] = 0.f;
        }
        issue_order();
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            f32x16 x[D / 32];
#pragma unroll
            for (int c = 0; c < D / 32; ++c) x[c] = splat16(0.f);
            if (word) cross_add_fine<TL>(TL::columns((t ? tq : tg) + same, at), t ? ds : p, x);
            cross_store<D>(x, t ? a.scale : 1.f, reinterpret_cast<float*>(tk), 0, l, [&](int row, int j, float (&v)[D / 8]) {
                if (k0 + row < a.Lk) cross_put<T, D>((t ? ok : ov) + (k0 + row) * (t ? a.dk : a.dv).row, j, v);
            });
            issue_order();
        }
    });
    __syncthreads();  // the tiles are done with
    float v[D / 8];
    merge_waves<D>(dq, reinterpret_cast<float*>(lds), tid, v);
    const int row = tid >> 3, j = tid & 7;
    if (row >= a.rows) return;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) v[i] *= a.scale;
    if (a.splits > 1) cross_leave<D>(a.part + it.slot(a, a.rows, 0) * (32 * D), row, j, v);
    else cross_put<T, D>(a.row(a.dq, it.b, it.g, row), j, v);
}

// -------------------------------------------------------------------------------------------------
// Backward, keys: dK and dV
// -------------------------------------------------------------------------------------------------
// The strip's keys are the lanes: what a key that is left out holds reaches its own lane only, whose results are zeros.
// The stage's rows' -lse and -D; rows behind the last have P = 0.
template <int ROWS>
struct CrossRowStats {
    const float *lse, *delta;
    float* lds;  // [2][2][64]
    int rows, tid;
    float e = 0.f, d = 0.f;
    __device__ __forceinline__ void load(int first) {
        if (tid < ROWS) {
            const bool there = first + tid < rows;
            e = there ? -lse[first + tid] : -__builtin_inff();
            d = there ? -delta[first + tid] : 0.f;
        }
    }
    __device__ __forceinline__ void store(int parity) {
        if (tid < ROWS) {
            lds[128 * parity + tid] = e;
            lds[128 * parity + 64 + tid] = d;
        }
    }
};

// The column pass's products with a tile of the stage, whose operands are read as they are needed: `row`, `col` are the lane's places for the first
// 16 features of a row and the first 32 columns, from which the others differ in bits, and are made anew each time (kept, they would be
// 24 registers at D = 128).
template <int D>
__device__ __forceinline__ f32x16 cross_feat(const char* t, int row, const typename BiasTile<__bf16, D>::Row& b, f32x16 acc) {
    asm volatile("" : "+v"(row));
#pragma unroll
    for (int i = 0; i < D / 16; ++i) acc = mfma_bf16(__builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(t + (row ^ 16 * i))), b.x[0][i], acc);
    return acc;
}
template <int D, bool FINE>
__device__ __forceinline__ void cross_add_t(const char* t, const int (&col)[2], float (&p)[16], f32x16 (&out)[D / 32]) {
    typedef s16x4 __attribute__((address_space(3))) * lds_ptr;
    int at[2] = {col[0], col[1]};
    asm volatile("" : "+v"(at[0]), "+v"(at[1]));
    bf16x8 w[2], rest[2];
    pack16(p, w);
    if (FINE) {
        cross_rest(p);
        pack16(p, rest);
    }
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(t + (at[0] ^ 64 * c) + 16 * i * BiasTile<__bf16, D>::ROW));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(t + (at[1] ^ 64 * c) + 16 * i * BiasTile<__bf16, D>::ROW));
            const bf16x8 x = __builtin_shufflevector(__builtin_bit_cast(bf16x4, lo), __builtin_bit_cast(bf16x4, hi), 0, 1, 2, 3, 4, 5, 6, 7);
            out[c] = mfma_bf16(x, w[i], out[c]);
            if (FINE) out[c] = mfma_bf16(x, rest[i], out[c]);
        }
}
// Wavefronts a SIMD.  Of bf16, D = 128, dK and dV are 128 registers beside the 64 of K and V; what is left of 256 is enough if nothing else is kept
// (2 x 16 heads over 4 of 2048 x 8192: 711 us with one wavefront and operands read ahead, 556 with two).  D = 64: 256 heads of 2048 x 2048 take 705 us
// with two, 656 with three.
template <class T, int D>
constexpr int cross_col_waves() { return sizeof(T) == 2 ? (D == 32 ? 4 : D == 64 ? 3 : 2) : D == 32 ? 2 : 1; }
template <class T, int D, bool FINE>
__global__ __launch_bounds__(256, (cross_col_waves<T, D>())) void cross_backward_col_kernel(CrossCall a) {
    typedef BiasTile<T, D> TL;
    typedef CrossStage<T, D> ST;
    constexpr int SUBS = ST::SUBS;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    CrossLds& sc = *reinterpret_cast<CrossLds*>(lds + cross_stages_bytes<T, D>());
    float* stats = reinterpret_cast<float*>(lds + cross_stages_bytes<T, D>() + sizeof(CrossLds));
    const int tid = threadIdx.x, w = uniform(tid >> 6), l = tid & 63, li = l & 31, h = l >> 5;
    const CrossItem it(a, gridDim.x);
    const int k0 = it.strip * 128 + 32 * w, ki = min(k0 + li, a.Lk - 1);
    const bool key = cross_key(a, it.b, k0 + li), some = __any(key);  // false behind the last key
    const typename TL::Row k = TL::load(a.k.head(it.b, it.g) + ki * a.k.row, h, k0 + li < a.Lk);
    const typename TL::Row v = TL::load(a.v.head(it.b, it.g) + ki * a.v.row, h, k0 + li < a.Lk);
    const typename TL::At at = TL::at(l);
    const float c2 = a.scale * LOG2E;
    f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) dk[c] = dv[c] = splat16(0.f);
    CrossRowStats<ST::ROWS> rs{a.lse + (size_t)it.bg * a.rows, a.delta + (size_t)it.bg * a.rows, stats, a.rows, tid};
    k.settled();
    v.settled();
    typedef CrossSource<T, D, false> S;
    // -lse or -D of a tile's rows
    auto stat = [&](const float* st) __attribute__((always_inline)) {
        f32x16 x;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 d = *reinterpret_cast<const f32x4*>(st + 8 * g);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * g + j] = d[j];
        }
        return x;
    };
    if (l == 0) sc.seg[w] = some;
    __syncthreads();
    if (sc.seg[0] | sc.seg[1] | sc.seg[2] | sc.seg[3])
        cross_walk<T, D, false>(a, sc, it, S(a, a.q, it.b, it.g), S(a, a.dout, it.b, it.g), lds, tid, rs,
            [&](const unsigned (&word)[SUBS], const char* buf, auto which) __attribute__((always_inline)) {
                if (!some) return;
#pragma unroll
                for (int u = 0; u < SUBS; ++u) {
                    if (word[u] == 0) continue;
                    const char *tq = buf + u * TL::BYTES, *tg = buf + (SUBS + u) * TL::BYTES;
                    const float* st = stats + 128 * which + 32 * u + 4 * h;
                    float x[16];  // P, then dS
                    if constexpr (sizeof(T) == 2) {
                        issue_order();
                        const f32x16 s = cross_feat<D>(tq, at.row[0], k, splat16(0.f));
                        issue_order();
                        const f32x16 e = stat(st);
#pragma unroll
                        for (int r = 0; r < 16; ++r) x[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c2, e[r]));
                        issue_order();
                        cross_add_t<D, false>(tg, at.col[0], x, dv);
                        issue_order();
                        const f32x16 dp = cross_feat<D>(tg, at.row[0], v, stat(st + 64));  // dP - D
                        issue_order();
#pragma unroll
                        for (int r = 0; r < 16; ++r) x[r] *= dp[r];
                        cross_add_t<D, FINE>(tq, at.col[0], x, dk);
                        issue_order();
                    } else {
                        const f32x16 s = TL::feat(TL::rows(tq, at), k);
                        if (D == 128) issue_order();
                        const f32x16 dp = TL::feat(TL::rows(tg, at), v, stat(st + 64));
                        if (D == 128) issue_order();
                        const f32x16 e = stat(st);
#pragma unroll
                        for (int r = 0; r < 16; ++r) x[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c2, e[r]));
                        TL::add_t(TL::columns(tg, at), x, dv);
#pragma unroll
                        for (int r = 0; r < 16; ++r) x[r] *= dp[r];
                        TL::add_t(TL::columns(tq, at), x, dk);
                    }
                }
            });
    __syncthreads();  // the stages are done with
    if (k0 >= a.Lk) return;
    const unsigned keys = (unsigned)__ballot(key);
    float* red = reinterpret_cast<float*>(lds);
    float* slot = a.part + it.slot(a, a.Lk, k0) * (2 * 32 * D);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        cross_store<D>(t ? dk : dv, t ? a.scale : 1.f, red, w, l, [&](int row, int j, float (&x)[D / 8]) {
            if (k0 + row >= a.Lk) return;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) x[i] = (keys >> row) & 1u ? x[i] : 0.f;
            if (a.splits > 1) cross_leave<D>(slot + t * 32 * D, row, j, x);
            else cross_put<T, D>((t ? a.dk : a.dv).head(it.b, it.g) + (k0 + row) * (t ? a.dk : a.dv).row, j, x);
        });
    }
}

// Strips of 32 keys, and a work-group's wavefronts take every fourth tile of the rows.
template <class T, int D>
constexpr int cross_col_few_bytes() { return cross_tiles_bytes<T, D>() + cross_shared_bytes<T, D>() + 4 * 64 * 4; }
template <class T, int D>
__global__ __launch_bounds__(256, (cross_backward_waves<T, D>())) void cross_backward_col_few_kernel(CrossCall a) {
    typedef BiasTile<T, D> TL;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, w = uniform(tid >> 6), l = tid & 63, li = l & 31, h = l >> 5;
    constexpr int TILES = cross_own_tiles<T, D>();
    char* const shared = lds + cross_tiles_bytes<T, D>();
    float* const stats = reinterpret_cast<float*>(shared + cross_shared_bytes<T, D>()) + 64 * w;
    const CrossItem it(a, gridDim.x);
    const int k0 = it.strip * 32, ki = min(k0 + li, a.Lk - 1);
    const bool key = cross_key(a, it.b, k0 + li);
    typename TL::Row k, v;
    if constexpr (TILES == 1) {
        typedef CrossSource<T, D, true> S;
        cross_share<T, D>(shared, S(a, a.k, it.b, it.g), S(a, a.v, it.b, it.g), k0, a.Lk, w, l);
    } else {
        k = TL::load(a.k.head(it.b, it.g) + ki * a.k.row, h, k0 + li < a.Lk);
        v = TL::load(a.v.head(it.b, it.g) + ki * a.v.row, h, k0 + li < a.Lk);
        k.settled();
        v.settled();
    }
    const typename TL::At at = TL::at(l);
    char* const tq = lds + w * TILES * TL::BYTES;
    char* const tg = tq + (TILES - 1) * TL::BYTES;
    const float c2 = a.scale * LOG2E;
    f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) dk[c] = dv[c] = splat16(0.f);
    typedef CrossSource<T, D, false> S;
    const S qs(a, a.q, it.b, it.g), gs(a, a.dout, it.b, it.g);
    const float *lse = a.lse + (size_t)it.bg * a.rows, *delta = a.delta + (size_t)it.bg * a.rows;
    const int tiles = __any(key) ? (a.rows + 31) / 32 : 0, step = 4 * a.splits;
    RowsInFlight<T, D> fq, other;
    RowsInFlight<T, D>& fg = TILES == 1 ? fq : other;  // (one tensor in flight, as in cross_few_walk)
    float e = 0.f, d = 0.f;
    auto fetch = [&](int tile) __attribute__((always_inline)) {
        fq.load(qs, tile * 32, l);
        if (TILES == 2) fg.load(gs, tile * 32, l);
        const int r = min(tile * 32 + li, a.rows - 1);
        e = lse[r], d = delta[r];
    };
    int tile = 4 * it.split + w;
    if (tile < tiles) fetch(tile);
    for (; tile < tiles; tile += step) {
        const unsigned word = tail_word(a.rows - tile * 32);
        const bool there = (word >> li) & 1u;
        const bool more = tile + step < tiles;
        auto put = [&](auto& rows, char* to) __attribute__((always_inline)) {
            wave_lds_order();
            rows.store(to, word, l);
            wave_lds_order();
        };
        if (l < 32) {
            stats[li] = there ? -e : -__builtin_inff();  // (rows behind the last have P = 0)
            stats[32 + li] = there ? -d : 0.f;
        }
        put(fq, tq);
        if (TILES == 2) {
            put(fg, tg);
            if (more) fetch(tile + step);
        }
        const float* const st = stats + 4 * h;
        auto stat = [&](int first) __attribute__((always_inline)) {
            f32x16 y;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(st + first + 8 * g);
#pragma unroll
                for (int j = 0; j < 4; ++j) y[4 * g + j] = x[j];
            }
            return y;
        };
        f32x16 s, dp;
        int same = 0;
        asm volatile("" : "+v"(same));
        if constexpr (TILES == 1) {
            fg.load(gs, tile * 32, l);
            s = TL::feat(TL::rows(tq, at), TL::rows(shared + same, at));
            issue_order();
            put(fg, tg);
            fq.load(qs, tile * 32, l);  // (once more, for dK)
            dp = TL::feat(TL::rows(tg, at), TL::rows(shared + TL::BYTES + same, at), stat(32));  // dP - D
            issue_order();
        } else {
            const f32x16 minus_d = stat(32);
            const typename TL::Row qr = TL::rows(tq, at), gr = TL::rows(tg, at);
            issue_order();
            s = TL::feat(qr, k);
            dp = TL::feat(gr, v, minus_d);
        }
        const f32x16 minus_lse = stat(0);
        float p[16], ds[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            p[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c2, minus_lse[r]));
            ds[r] = p[r] * dp[r];
        }
        cross_add_fine<TL>(TL::columns(tg, at), p, dv);
        if (TILES == 1) {
            put(fq, tq);
            if (more) fetch(tile + step);
        }
        cross_add_fine<TL>(TL::columns(tq, at), ds, dk);
    }
    const unsigned keys = (unsigned)__ballot(key);
    const int row = tid >> 3, j = tid & 7;
    const bool keep = (keys >> row) & 1u;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        __syncthreads();  // the tiles, and what was there before, are done with
        float x[D / 8];
        merge_waves<D>(t ? dk : dv, reinterpret_cast<float*>(lds), tid, x);
        if (k0 + row >= a.Lk) continue;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) x[i] = keep ? x[i] * (t ? a.scale : 1.f) : 0.f;
        if (a.splits > 1) cross_leave<D>(a.part + it.slot(a, a.Lk, k0) * (2 * 32 * D) + t * 32 * D, row, j, x);
        else cross_put<T, D>((t ? a.dk : a.dv).head(it.b, it.g) + (k0 + row) * (t ? a.dk : a.dv).row, j, x);
    }
}

template <class T, int D, bool MANY>
__global__ __launch_bounds__(256) void cross_merge_col_kernel(CrossCall a) {
    typedef CrossJoin<D, MANY> J;
    __shared__ f32x4 red[2][MANY ? 256 : 1];
    const int tid = threadIdx.x;
    const J j(tid);
    const int sets = (a.Lk + J::ROWS - 1) / J::ROWS, bg = blockIdx.x / sets, key = min((int)(blockIdx.x - bg * sets) * J::ROWS + j.row, a.Lk - 1);
    const float* slot = a.part + ((size_t)bg * ((a.Lk + 31) / 32) + key / 32) * a.splits * (2 * 32 * D) + (key % 32) * D;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const f32x4 x = j.sum(slot + t * 32 * D, a.splits, 2 * 32 * D, red[t], [](int) { return 1.f; });
        const HeadsAt& to = t ? a.dk : a.dv;
        if (j.group == 0) cross_put4<T>(to.head(bg / a.G, bg % a.G) + key * to.row, j.col, x);
    }
}

}  // namespace spion

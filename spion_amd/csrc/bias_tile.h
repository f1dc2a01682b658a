// What the kernels of the attention with a relative position bias share (bias_kernels.h): 32 x D tiles in LDS for bf16 and fp32
// and the matrix operands read from them, the bias table of a head, and the list of the tiles a strip has to visit.
#pragma once
#include "bf16_kernels.h"

namespace spion {

// Heads of one tensor, [B][H][L][D] by strides in bytes.
struct HeadsAt {
    const char* p;
    long long b, h, row;
    __device__ __forceinline__ const char* head(int ib, int ih) const { return p + ib * b + ih * h; }
};
// One head: its buffer, the bytes from row to row.  A head lies within 2^31 bytes and its rows 2^24 apart at most, so the offsets
// of rows up to 64 behind its end still count; what lies behind the buffer reads as zeros.
struct HeadBuf {
    rsrc_t r;
    int ld;
    template <class T, int D>
    __device__ static __forceinline__ HeadBuf of(const HeadsAt& t, int b, int h, int rows) {
        // (the same in every lane, which the compiler does not see through the divisions that b and h come from)
        const unsigned long long p = reinterpret_cast<unsigned long long>(t.head(b, h));
        const unsigned long long q = (unsigned)uniform((int)(unsigned)p) | (unsigned long long)(unsigned)uniform((int)(p >> 32)) << 32;
        return HeadBuf{make_rsrc(reinterpret_cast<const void*>(q), (unsigned)((rows - 1) * t.row + D * (int)sizeof(T))), (int)t.row};
    }
    __device__ __forceinline__ int at(int row, int byte) const { return (int)((unsigned)row * (unsigned)ld + (unsigned)byte); }
};

struct BiasCall {
    HeadsAt q, k, v, o, dout, dq, dk, dv;
    const void* w;      // [buckets][H], of the heads' type
    const int* map;     // [2 R + 1]: bucket of every difference -R .. R
    const void* mask;   // [B][Lk]: null, float (0 = left out) or bytes
    const float* mat;   // [nb][nb] pattern of bs x bs blocks, or null
    float* lse;         // [B*H][Lq]: log2 of the softmax denominator, +inf for rows that nothing enters (NaN stays NaN)
    float* delta;       // [B*H][Lq]: sum over the keys of P dP
    float* part;        // workspace: the pieces' slots
    float* tables;      // workspace: the table's gradient by strips, [B*H][strips][splits][buckets]
    float* mean;        // [Lq][Lk]
    int B, H, Lq, Lk, R, buckets, off, bs, nb;
    int mask_bytes;     // 4 or 1
    int strips, splits, per_split;  // strips of 32 (or 128) rows, pieces of the other side, tiles of 32 to a piece
    int strips32;                   // strips of 32 rows
    float scale;
};

// ---------------------------------------------------------------------------------------------------------------------
// 32 x D tiles
// ---------------------------------------------------------------------------------------------------------------------
// A tile in LDS is one bf16 image, or three for fp32 heads: every value as the sum of three bf16 numbers, split by the thread that
// stages it (Split3 in tile_ops.h: six products of the parts give fp32 accuracy at 2.7 times the rate of the fp32 matrix
// instructions; an infinite operand, or one of 2^127 and more, makes sums that it enters NaN).  Rows are stored as 16-byte pieces of
// eight values, piece c of row r at c ^ swz(r): sixteen rows' reads of one piece, and the transposing reads of four rows, meet every
// bank once.
//   rows()   lane (li, h) has features h*D/2 .. of row li, the operand of a product over the head dimension
//   columns(), add_t()  out[c] += X^T . W, W given as the accumulator values of a 32 x 32 product whose rows are the tile's rows; the
//            accumulator layout is then the other operand's, register for register after conversion.  With bf16 heads W's rounding
//            is off by up to 2^-8 of each weight, as the outputs' own is; sums are fp32.
template <class T, int D>
struct BiasTile {
    static constexpr int IM = sizeof(T) == 4 ? 3 : 1;
    // Whether the transposed operands are read ahead of the arithmetic that they come after: three images of them are too many registers.
    static constexpr bool EARLY = IM == 1;
    static constexpr int ROW = D * 2, IMAGE = 32 * ROW, BYTES = IM * IMAGE, CPR = D / 8;
    struct Row {
        bf16x8 x[IM][D / 16];
        // its loads waited for: else the compiler waits at the first use inside the walk, for the tiles just asked for as well
        __device__ __forceinline__ void settled() const {
#pragma unroll
            for (int m = 0; m < IM; ++m) settle(x[m]);
        }
    };
    struct Columns {
        bf16x8 x[IM][D / 32][2];
    };
    struct At {
        int row[D / 16], col[D / 32][2];
    };
    __device__ static __forceinline__ int swz(int r) {
        if constexpr (D == 64) return ((r << 1) & 4) | ((r >> 1) & 2) | ((r >> 3) & 1);  // even (odd) rows of 16: all eight, r and r + 2 differ in 4
        else return (r >> 2) & 3;
    }
    __device__ static __forceinline__ At at(int l) {
        const int li = l & 31, h = l >> 5, gm = (l >> 4) & 1, j = l & 15, r = 4 * h + (j >> 2);
        At a;
#pragma unroll
        for (int t = 0; t < D / 16; ++t) a.row[t] = li * ROW + 16 * ((h * (CPR / 2) + t) ^ swz(li));
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
            for (int u = 0; u < 2; ++u)
                a.col[c][u] = (r + 8 * u) * ROW + 16 * ((4 * c + 2 * gm + ((j & 3) >> 1)) ^ swz(r + 8 * u)) + 8 * (j & 1);
        return a;
    }
    __device__ static __forceinline__ Row rows(const char* t, const At& a) {
        Row r;
#pragma unroll
        for (int m = 0; m < IM; ++m)
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
                r.x[m][i] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(t + m * IMAGE + a.row[i]));
        return r;
    }
    // eight values from memory, split
    __device__ static __forceinline__ void split_piece(const char* p, u32x4 (&x)[IM]) {
        if constexpr (IM == 1) {
            x[0] = *reinterpret_cast<const u32x4*>(p);
        } else {
            split_values(*reinterpret_cast<const f32x4*>(p), *reinterpret_cast<const f32x4*>(p + 16), x);
        }
    }
    __device__ static __forceinline__ void split_values(f32x4 a, f32x4 b, u32x4 (&x)[IM]) {
        const float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        const Split3<8> s = split3(v);
#pragma unroll
        for (int m = 0; m < IM; ++m) x[m] = __builtin_bit_cast(u32x4, s.p[m][0]);
    }
    // row `row` of a head, from global memory; zeros where `there` is false
    __device__ static __forceinline__ Row load(const char* row, int h, bool there) {
        Row r;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            u32x4 v[IM];
#pragma unroll
            for (int m = 0; m < IM; ++m) v[m] = u32x4{0, 0, 0, 0};
            if (there) split_piece(row + (h * (D / 2) + 8 * i) * sizeof(T), v);
#pragma unroll
            for (int m = 0; m < IM; ++m) r.x[m][i] = __builtin_bit_cast(bf16x8, v[m]);
        }
        return r;
    }
    __device__ static __forceinline__ float value(const Row& r, int i, int e) {
        float v = (float)r.x[0][i][e];
        if constexpr (IM == 3) v += (float)r.x[1][i][e] + (float)r.x[2][i][e];
        return v;
    }
    __device__ static __forceinline__ float dot(const Row& a, const Row& b) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fmaf(value(a, i, e), value(b, i, e), s);
        return s;
    }
    __device__ static __forceinline__ f32x16 feat(const Row& a, const Row& b, f32x16 acc = splat16(0.f)) {
        if constexpr (IM == 3) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                acc = mfma_bf16(a.x[2][i], b.x[0][i], acc);
                acc = mfma_bf16(a.x[0][i], b.x[2][i], acc);
                acc = mfma_bf16(a.x[1][i], b.x[1][i], acc);
                acc = mfma_bf16(a.x[1][i], b.x[0][i], acc);
                acc = mfma_bf16(a.x[0][i], b.x[1][i], acc);
            }
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) acc = mfma_bf16(a.x[0][i], b.x[0][i], acc);
        return acc;
    }
    // the tile feature-major, with the transposing LDS read
    __device__ static __forceinline__ Columns columns(const char* t, const At& a) {
        Columns xt;
        typedef s16x4 __attribute__((address_space(3))) * lds_ptr;
#pragma unroll
        for (int m = 0; m < IM; ++m)
#pragma unroll
            for (int c = 0; c < D / 32; ++c)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(t + m * IMAGE + a.col[c][0] + 16 * i * ROW));
                    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(t + m * IMAGE + a.col[c][1] + 16 * i * ROW));
                    xt.x[m][c][i] = __builtin_shufflevector(__builtin_bit_cast(bf16x4, lo), __builtin_bit_cast(bf16x4, hi), 0, 1, 2, 3, 4, 5, 6, 7);
                }
        return xt;
    }
    __device__ static __forceinline__ void add_t(const Columns& xt, const float (&p)[16], f32x16 (&out)[D / 32]) {
        if constexpr (IM == 1) {
            bf16x8 wb[2];
            pack16(p, wb);
            mma_tile_bf16<D>(xt.x[0], wb, out);
        } else {
            const Split3<16> w = split3(p);
            constexpr int PAIRS[6][2] = {{2, 0}, {0, 2}, {1, 1}, {1, 0}, {0, 1}, {0, 0}};
#pragma unroll
            for (int k = 0; k < 6; ++k) mma_tile_bf16<D>(xt.x[PAIRS[k][0]], w.p[PAIRS[k][1]], out);
        }
    }
};

// Eight values on their way from global memory to LDS.
template <class T>
struct PieceInFlight {
    u32x4 x[sizeof(T) / 2];
    __device__ __forceinline__ void load(rsrc_t r, int at) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) x[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at + 16 * i, 0, 0));
    }
    // piece c of row r of tile t; a row that is left out becomes zeros (whatever lies in it: 0 times it is 0)
    template <int D, bool ALL>
    __device__ __forceinline__ void store(char* t, int r, int c, bool there) const {
        typedef BiasTile<T, D> TL;
        u32x4 v[TL::IM];
        if constexpr (TL::IM == 1) v[0] = x[0];
        else TL::split_values(__builtin_bit_cast(f32x4, x[0]), __builtin_bit_cast(f32x4, x[1]), v);
#pragma unroll
        for (int m = 0; m < TL::IM; ++m) {
            if (!ALL && !there) v[m] = u32x4{0, 0, 0, 0};
            *reinterpret_cast<u32x4*>(t + m * TL::IMAGE + r * TL::ROW + 16 * (c ^ TL::swz(r))) = v[m];
        }
    }
};

// A wavefront's tile on its way from global memory to LDS: piece n = 64 i + l of the tile is piece n % CPR of row n / CPR.
template <class T, int D>
struct TileInFlight {
    typedef BiasTile<T, D> TL;
    static constexpr int N = TL::CPR / 2;
    PieceInFlight<T> x[N];
    // rows first .. first + 31
    __device__ __forceinline__ void load(const HeadBuf& head, int first, int l) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int n = 64 * i + l, r = n / TL::CPR, c = n % TL::CPR;
            x[i].load(head.r, head.at(first, head.at(r, 8 * c * (int)sizeof(T))));
        }
    }
    // to LDS; rows whose bit of `word` is not set are left out
    __device__ __forceinline__ void store(char* t, unsigned word, int l) const {
        if (word == ~0u) put<true>(t, word, l);
        else put<false>(t, word, l);
    }
    template <bool ALL>
    __device__ __forceinline__ void put(char* t, unsigned word, int l) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int n = 64 * i + l, r = n / TL::CPR, c = n % TL::CPR;
            x[i].template store<D, ALL>(t, r, c, (word >> r) & 1u);
        }
    }
};

// What stands before is issued before what follows: LDS reads ahead of the arithmetic whose operands they are not, which the
// compiler would move to their use, one register set and one full latency at a time.
__device__ __forceinline__ void issue_order() { __builtin_amdgcn_sched_barrier(0); }

// READS LDS reads issued between PRODUCTS matrix instructions that stand in the same block.
template <int PRODUCTS, int READS>
__device__ __forceinline__ void read_behind_products() {
#pragma unroll
    for (int i = 0; i < PRODUCTS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS / PRODUCTS, 0);
    }
}

// Orders a wavefront's own LDS accesses (they complete in order; this is for the compiler).
__device__ __forceinline__ void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// ---------------------------------------------------------------------------------------------------------------------
// The bias
// ---------------------------------------------------------------------------------------------------------------------
// A head's bias by position difference, log2 domain: entry i is difference i - R - BIAS_PAD; differences beyond R on either
// side have the outermost buckets.  The padding is what tiles that touch (-R, R) reach beyond it (62), so their look-ups need
// no clamping; tiles further out take one number for all their pairs.
constexpr int BIAS_PAD = 64;
__host__ __device__ inline int bias_entries(int R) { return 2 * (R + BIAS_PAD) + 1; }
__host__ __device__ inline int bias_floats(int R) { return (bias_entries(R) + 3) & ~3; }

__device__ __forceinline__ int bucket_at(const BiasCall& a, int diff) {
    const int k = a.map[min(max(diff, -a.R), a.R) + a.R];
    return min(max(k, 0), a.buckets - 1);
}
template <class T>
__device__ __forceinline__ float bias_weight(const BiasCall& a, int bucket, int h) {
    return (float)reinterpret_cast<const T*>(a.w)[(size_t)bucket * a.H + h] * LOG2E;
}
// The table, and with `buckets` what bucket each entry is of.
template <class T>
__device__ __forceinline__ void fill_bias(const BiasCall& a, int h, float* tab, int tid, unsigned short* buckets = nullptr) {
#pragma unroll 2
    for (int i = tid; i < bias_entries(a.R); i += 256) {
        const int k = bucket_at(a, i - a.R - BIAS_PAD);
        tab[i] = bias_weight<T>(a, k, h);
        if (buckets) buckets[i] = (unsigned short)k;
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Tiles to visit
// ---------------------------------------------------------------------------------------------------------------------
// The other side of a strip is walked in chunks of CHUNK tiles of 32.  For a chunk the work-group makes, in LDS, the list of
// the tiles that the strip has to visit, in order: those of the pattern that have a key which takes part.  words: which keys of
// each tile do.  Everything is read from the mask and the pattern as they are at the call.
constexpr int CHUNK = 512;
struct ScanLds {
    unsigned words[CHUNK];
    unsigned short list[CHUNK];
    int seg[8], pat[8];
    unsigned char who[CHUNK];  // of stages: which wavefronts' rows have them in their pattern
    int pats[4][8];
    float ml[4][2][32];
    float row[32];
};
static_assert(sizeof(ScanLds) % 16 == 0, "what follows it is aligned");

__device__ __forceinline__ bool key_there(const BiasCall& a, int b, int key) {
    if (key >= a.Lk) return false;
    if (a.mask == nullptr) return true;
    const size_t i = (size_t)b * a.Lk + key;
    return a.mask_bytes == 4 ? reinterpret_cast<const float*>(a.mask)[i] != 0.f : reinterpret_cast<const unsigned char*>(a.mask)[i] != 0;
}

// Which of the 32 keys of a tile there are, without a mask.
__device__ __forceinline__ unsigned tail_word(int left) { return left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1u; }

// Words of groups of 64 keys, w, w + 4, ... of n, from a mask: eight groups' loads are on their way together.
template <class M>
__device__ __forceinline__ void mask_words(const M* mask, unsigned* words, int first, int n, int keys, int w, int l) {
    constexpr int AHEAD = 8;
    for (int g0 = w; g0 < n; g0 += 4 * AHEAD) {
        M x[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) x[u] = mask[min((first + 2 * (g0 + 4 * u)) * 32 + l, keys - 1)];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int g = g0 + 4 * u;
            const unsigned long long there = __ballot(x[u] != (M)0 && (first + 2 * g) * 32 + l < keys);
            if (l == 0 && g < n) {
                words[2 * g] = (unsigned)there;
                if (2 * g + 1 < CHUNK) words[2 * g + 1] = (unsigned)(there >> 32);
            }
        }
    }
}

// Which keys of tiles first .. first + count - 1 there are.
__device__ __forceinline__ void scan_words(const BiasCall& a, ScanLds& s, int b, int first, int count, int tid) {
    const int w = uniform(tid >> 6), l = tid & 63;
    if (a.mask) {
        const size_t row = (size_t)b * a.Lk;
        if (a.mask_bytes == 4) mask_words(reinterpret_cast<const float*>(a.mask) + row, s.words, first, (count + 1) / 2, a.Lk, w, l);
        else mask_words(reinterpret_cast<const unsigned char*>(a.mask) + row, s.words, first, (count + 1) / 2, a.Lk, w, l);
    } else {
        for (int i = tid; i < CHUNK; i += 256) s.words[i] = i < count ? tail_word(a.Lk - (first + i) * 32) : 0;
    }
    __syncthreads();
}

// Tiles first .. first + count - 1 (count <= CHUNK) of the other side, for strip `own` of 32 rows.  KEYS: the other side is the
// keys, else the queries.  Returns how many are listed; in_pattern grows by the keys of the pattern's tiles.  All threads of
// the work-group call it; LDS that they still read must be done with.
template <bool KEYS>
__device__ __forceinline__ int scan_chunk(const BiasCall& a, ScanLds& s, int b, int own, int first, int count, int tid,
                                          int& in_pattern) {
    const int w = uniform(tid >> 6), l = tid & 63;
    __syncthreads();
    if (KEYS) scan_words(a, s, b, first, count, tid);
    bool act[2];
    unsigned long long votes[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int i = tid + 256 * r, tile = first + i;
        bool in = i < count;
        if (in && a.mat) {
            const int o = own * 32 / a.bs, t = tile * 32 / a.bs;
            in = a.mat[KEYS ? (size_t)o * a.nb + t : (size_t)t * a.nb + o] != 0.f;
        }
        const unsigned long long pat = __ballot(in);
        const unsigned long long tail = KEYS ? __ballot(in && tile * 32 + 32 > a.Lk) : 0;
        act[r] = in && (!KEYS || s.words[i] != 0);
        votes[r] = __ballot(act[r]);
        if (l == 0) {
            s.seg[4 * r + w] = __popcll(votes[r]);
            s.pat[4 * r + w] = 32 * __popcll(pat) - (tail ? 32 - (a.Lk & 31) : 0);
        }
    }
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        int before = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) before += k < 4 * r + w ? s.seg[k] : 0;
        if (act[r]) s.list[before + __popcll(votes[r] & ((1ull << l) - 1))] = (unsigned short)(tid + 256 * r);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        total += s.seg[k];
        in_pattern += s.pat[k];
    }
    __syncthreads();
    return total;
}

// Wavefronts' 32 x D results acc[c][r] (lane (li, h): row li, feature 32 c + acc_row(r, h)) added up in the wavefronts' order in LDS
// (4 x 32 x (D + 4) floats).  Afterwards thread t has the sums of features 8 j .. of row t / 8, j = t % 8 + 8 n, in x[n].
template <int D>
constexpr int merge_floats() { return 4 * 32 * (D + 4); }
template <int D>
__device__ __forceinline__ void merge_waves(const f32x16 (&acc)[D / 32], float* red, int tid, float (&x)[D / 8]) {
    const int w = uniform(tid >> 6), l = tid & 63, li = l & 31, h = l >> 5;
    float* mine = red + (w * 32 + li) * (D + 4);
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<f32x4*>(mine + 32 * c + 8 * g + 4 * h) =
                f32x4{acc[c][4 * g], acc[c][4 * g + 1], acc[c][4 * g + 2], acc[c][4 * g + 3]};
    __syncthreads();
    const int row = tid >> 3, j = tid & 7;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) x[i] = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(red + (k * 32 + row) * (D + 4) + j * (D / 8) + 4 * i);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * i + e] += v[e];
        }
}
// D / 8 consecutive values to memory, rounded once
template <class T, int N>
__device__ __forceinline__ void store_values(char* p, const float (&x)[N]) {
    T* t = reinterpret_cast<T*>(p);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) *reinterpret_cast<f32x4*>(t + 4 * i) = f32x4{x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            bf16x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (__bf16)x[4 * i + e];
            *reinterpret_cast<bf16x4*>(t + 4 * i) = v;
        }
    }
}

}  // namespace spion

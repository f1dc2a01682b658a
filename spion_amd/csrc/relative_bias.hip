// Host side of the attention with a learned bias by buckets of relative position (kernels: bias_kernels.h): argument checks,
// launch shapes, workspaces.  No handle: sizes come with the call, and nothing is kept from one call for another.
#include "bias_dense_kernels.h"
#include "common.h"
#include "../../include/spion_hip.h"

#include <algorithm>
#include <climits>

namespace spion {

typedef spion_bias_attention Call;

static long long strips_of(int rows, int strip = 32) { return (rows + strip - 1) / strip; }
static int slot_floats(const Call& c) { return 32 * c.head_dim + 96; }  // bias_slot

// How one side of a call is walked: in strips of 128 or 64 rows over shared stages, or of 32 with the tiles dealt to the wavefronts,
// and the other side in `splits` pieces.
struct Walk {
    int rows;
    int strips, splits, per_split;  // tiles of 32 to a piece
    void cut(long long tiles, long long pieces, int unit) {
        const long long units = (tiles + unit - 1) / unit, each = (units + pieces - 1) / pieces;
        per_split = (int)(each * unit);
        splits = (int)((units + each - 1) / each);  // none of them empty
    }
};
// Which of the two, by what fills the machine.  A pattern goes in strips of 128 only with blocks that hold whole stages (64 x 64 and
// more; of smaller blocks the rows of a strip would have few in common), and so does a side of more than two tiles only.  (us below:
// strips of 32 against strips of 128; forward of L = 1024 unless said otherwise.)
//   bf16: strips of 128, uncut, once there is one for each CU (d = 64: 256 strips 28.4 / 24.4, 128 strips 16.1 / 24.0); the forward
//     and the row pass at d = 32, with half the arithmetic to a stage, from two for each CU (384: 24.2 / 25.6, 512: 29.4 / 25.7).
//     Cut in two to fill the machine, 128 strips take 22.8: the pieces' merge costs what they gain.
//   fp32, six products for one: fewer strips than the CUs hold are cut into pieces of at least 256 rows of the other side, and
//     strips of 32 stay for launches that leave a quarter of the CUs idle even so (d = 64, 192 strips of L = 320: 39.8 / 24.5), and
//     at d = 32 for the short ones among those that would have to be cut (128 strips: 24.7 / 27.3, of L = 4096 77.9 / 63.0).
// The number of pieces is the one with the least rounds of work-groups times tiles to a piece, and the cost of the pieces.  A CU holds one
// work-group of the fp32 backward at d = 64 (its LDS) and else two, which take 1.75 times as long together as one alone.  A merge
// (5 us) counts as 2 tiles and 6, and every round of work-groups past the first that the machine holds as 4 and 2.5: their sums are
// written and read again, and their tables set up.  (us, 12 heads of 1000, d = 64, backward: 1 / 2 / 4 pieces 163 / 129 / 142.  24
// heads of 2048 in 1 / 2 / 8 pieces: forward 167 / 157 / 173, backward 663 / 563 / 755, at d = 32 102 / 95 / 104 and 297 / 288 / 302; 34 heads
// 273 / 238 / 240, 994 / 901 / 1074, 166 / 142 / 142, 490 / 435 / 451; 257 heads 1467 / 1512 / 1855, 5744 / 6067 / 8130, 838 / 867 / 1048,
// 2641 / 2743 / 3482.)  No more than eight work-groups to a CU: what pieces leave in the workspace stays below 71 MB forward and 135
// backward at d = 64, half of it at 32; launches that fill the machine four times over are not cut, and could gain a tenth at most.
enum class Pass { FORWARD, ROW, COL };
static Walk walk_of(const Call& c, int rows, int others, bool can_split, Pass pass) {
    const long long cus = device_cus(), wide = (long long)c.batch * c.heads * strips_of(rows, 128), tiles = strips_of(others);
    long long pieces = 1;
    bool dense = (!c.mat || c.block_size % 64 == 0) && rows > 64;
    if (c.bf16) {
        dense = dense && wide >= (c.head_dim == 32 && pass != Pass::COL ? 2 * cus : cus);
    } else {
        const bool alone = c.head_dim == 64 && pass != Pass::FORWARD;
        double least = 0;
        for (long long n = 1; n == 1 || (can_split && n <= std::min(tiles / 8, 16LL) && n * wide <= 8 * cus); ++n) {
            const long long rounds = (wide * n + cus - 1) / cus, each = (tiles + n - 1) / n;
            const double all = (double)(wide * n) / cus;
            const double extra = n == 1 ? 0 : alone ? 2 + 4 * std::max(0., all - 1) : 6 + 2.5 * std::max(0., all - 2);
            const double cost = (alone ? (double)rounds : 1.75 * (rounds / 2) + rounds % 2) * each + extra;
            if (n == 1 || cost < least) least = cost, pieces = n;
        }
        dense = dense && 4 * wide * pieces >= 3 * cus && (c.head_dim == 64 || tiles > 32 || 4 * wide >= 3 * cus);
    }
    Walk w{};
    w.rows = dense ? 128 : 32;
    // Strips of 64 rows, uncut, two wavefronts to the same rows (fp32 heads of 64 features have no second tile in a stage for that): in
    // patterns of odd multiples of 64, where the rows of a strip of 128 lie in two block rows (16 heads of 8192, bf16, a tenth
    // of the blocks: 326 / 312), and in the column pass at d = 32, whose strips of 128 come in less than two rounds (bf16,
    // 384 strips of L = 1024 and 2048 75 / 67 and 113 / 99, 512 of 1024 79 / 89; fp32 184 / 165, 512 186 / 194).
    const bool halves = (c.bf16 || c.head_dim == 32) && rows > 64 && (!c.mat || c.block_size % 64 == 0);
    const bool odd = c.mat && c.block_size % 128 != 0 && (long long)c.batch * c.heads * strips_of(rows, 64) >= cus;
    const bool few = !c.mat && pass == Pass::COL && c.head_dim == 32 && 4 * wide >= 3 * cus && wide < 2 * cus;
    if (halves && (odd || few)) {
        w.rows = 64;
        pieces = 1;
        dense = true;
    }
    w.strips = (int)strips_of(rows, w.rows);
    w.cut(tiles, dense ? pieces : 1, dense ? 2 : 1);
    return w;
}
// The forward's strips of 32 rows go in pieces as well, each wavefront keeping at least two tiles.
static Walk forward_walk(const Call& c, bool can_split) {
    Walk w = walk_of(c, c.q_len, c.k_len, can_split, Pass::FORWARD);
    if (w.rows > 32 || !can_split) return w;
    const long long groups = (long long)c.batch * c.heads * w.strips, tiles = strips_of(c.k_len);
    w.cut(tiles, std::max(1LL, std::min({(2LL * device_cus() + groups - 1) / groups, tiles / 8, 64LL})), 1);
    return w;
}
// Pieces of the (head, sample) pairs that the mean map is added up in.
static int mean_splits(const Call& c) {
    const long long tiles = strips_of(c.q_len, 64) * strips_of(c.k_len, 64), pairs = (long long)c.batch * c.heads;
    return (int)std::max(1LL, std::min({4LL * device_cus() / tiles, pairs / 4, 16LL}));
}

static long long workspace_floats(const Call& c, bool backward) {
    const long long nb = (long long)c.batch * c.heads;
    if (backward) {
        const Walk row = walk_of(c, c.q_len, c.k_len, true, Pass::ROW), col = walk_of(c, c.k_len, c.q_len, true, Pass::COL);
        const long long a = row.splits > 1 ? nb * strips_of(c.q_len) * row.splits * slot_floats(c) : 0;
        const long long b = col.splits > 1 ? nb * strips_of(c.k_len) * col.splits * 64 * c.head_dim : 0;
        // D, rounded up to whole pieces of 16 bytes, the table's gradient by strips, alike, the pieces
        return ((nb * c.q_len + 3) & ~3LL) + ((nb * col.strips * col.splits * c.num_buckets + 3) & ~3LL) + std::max(a, b);
    }
    const Walk w = forward_walk(c, true);
    const int m = mean_splits(c);
    return std::max(w.splits > 1 ? nb * strips_of(c.q_len) * w.splits * slot_floats(c) : 0,
                    c.Mean && m > 1 ? (long long)m * c.q_len * c.k_len : 0);
}

// Work-groups of 256 threads that a launch holds (2^32 threads and more are refused by the runtime, in the middle of a call).
constexpr long long MOST_GROUPS = (1 << 24) - 1;

static bool sizes_ok(const char* who, const Call& c) {
    if (c.batch < 1 || c.heads < 1 || c.q_len < 1 || c.k_len < 1 || c.num_buckets < 1) {
        set_error("%s: sizes are positive", who);
        return false;
    }
    if (c.head_dim != 32 && c.head_dim != 64) {
        set_error("%s: head_dim %d, 32 or 64 expected", who, c.head_dim);
        return false;
    }
    if (c.max_distance < 1 || c.max_distance > SPION_BIAS_MAX_DISTANCE) {
        set_error("%s: max_distance %d, 1 to %d expected", who, c.max_distance, SPION_BIAS_MAX_DISTANCE);
        return false;
    }
    if (c.num_buckets > 32767) {
        set_error("%s: up to 32767 buckets", who);
        return false;
    }
    if (c.q_len > (1 << 29) || c.k_len > (1 << 29) || c.offset > (1 << 29) || c.offset < -(1 << 29)) {
        set_error("%s: lengths and offset up to 2^29", who);
        return false;
    }
    const long long longest = std::max(c.q_len, c.k_len);
    if ((long long)c.batch * c.heads > MOST_GROUPS || (long long)c.batch * c.heads * strips_of((int)longest) > MOST_GROUPS ||
        (long long)c.num_buckets * c.heads > MOST_GROUPS) {
        set_error("%s: too many heads and rows, or heads and buckets, for one launch", who);
        return false;
    }
    if (c.mat && (c.block_size < 32 || c.block_size % 32 || c.block_size > (1 << 29) || c.q_len != c.k_len || c.offset != 0)) {
        set_error("%s: a pattern has blocks of a multiple of 32 (%d) and as many queries as keys, without an offset", who,
                  c.block_size);
        return false;
    }
    if (c.key_mask && c.mask_bytes != 1 && c.mask_bytes != 4) {
        set_error("%s: a key mask has 1 or 4 bytes a key", who);
        return false;
    }
    return true;
}

static bool heads_ok(const char* who, const char* name, const Call& c, const spion_heads& t, int rows, bool written) {
    if (!t.p) {
        set_error("%s: null pointer (%s)", who, name);
        return false;
    }
    const int unit = c.bf16 ? 8 : 4;
    if (reinterpret_cast<uintptr_t>(t.p) % 16 || t.batch_stride % unit || t.head_stride % unit || t.row_stride % unit ||
        t.batch_stride < 0 || t.head_stride < 0 || t.row_stride < 0 || (written && t.row_stride < c.head_dim)) {
        set_error("%s: %s: 16-byte aligned heads with strides in multiples of 16 bytes expected", who, name);
        return false;
    }
    const int e = c.bf16 ? 2 : 4;
    if (t.row_stride > (1 << 24) / e || (rows - 1) * t.row_stride * e + c.head_dim * e > INT_MAX) {
        set_error("%s: %s: rows up to 2^24 bytes apart and heads within 2^31 bytes expected", who, name);
        return false;
    }
    return true;
}

static HeadsAt heads_at(const Call& c, const spion_heads& t) {
    const int e = c.bf16 ? 2 : 4;
    return HeadsAt{reinterpret_cast<const char*>(t.p), t.batch_stride * e, t.head_stride * e, t.row_stride * e};
}

static BiasCall device_call(const Call& c) {
    BiasCall a{};
    a.q = heads_at(c, c.Q), a.k = heads_at(c, c.K), a.v = heads_at(c, c.V), a.o = heads_at(c, c.Out);
    a.dout = heads_at(c, c.dO), a.dq = heads_at(c, c.dQ), a.dk = heads_at(c, c.dK), a.dv = heads_at(c, c.dV);
    a.w = c.weight, a.map = c.buckets, a.mask = c.key_mask, a.mat = c.mat;
    a.lse = c.Lse, a.mean = c.Mean;
    a.B = c.batch, a.H = c.heads, a.Lq = c.q_len, a.Lk = c.k_len, a.R = c.max_distance, a.buckets = c.num_buckets;
    a.off = c.offset, a.bs = c.block_size, a.nb = c.mat ? (c.k_len + c.block_size - 1) / c.block_size : 0;
    a.mask_bytes = c.mask_bytes;
    a.splits = 1;
    a.scale = 1.0f / sqrtf((float)c.head_dim);
    return a;
}

template <class K>
static bool launch(const char* name, K kernel, long long groups, size_t lds, hipStream_t stream, const BiasCall& a) {
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) {
            set_error("%s: %zu bytes of LDS: %s", name, lds, hipGetErrorString(e));
            return false;
        }
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(256), lds, stream, a);
    return check_launch(name);
}

template <class T, int D>
static size_t stages_lds(const BiasCall& a) {
    return bias_stages_bytes<T, D>() + bias_floats(a.R) * 4 + sizeof(ScanLds);
}
template <class T, int D>
static size_t walk_lds(const BiasCall& a) {
    return bias_tiles_bytes<T, D>() + bias_floats(a.R) * 4 + sizeof(ScanLds);
}
static void take(BiasCall& a, const Walk& w, int rows) {
    a.strips = w.strips;
    a.splits = w.splits;
    a.per_split = w.per_split;
    a.strips32 = (int)strips_of(rows);
}

template <class T, int D>
static bool forward(const Call& c, hipStream_t stream) {
    BiasCall a = device_call(c);
    const long long nb = (long long)a.B * a.H;
    const bool room = c.workspace && c.workspace_floats >= workspace_floats(c, false);
    const Walk w = forward_walk(c, room);
    take(a, w, a.Lq);
    a.part = c.workspace;
    const long long groups = nb * w.strips * w.splits;
    bool ok = true;
    if (w.rows == 128) ok = launch("bias_forward_dense_kernel", bias_forward_dense_kernel<T, D, true>, groups, stages_lds<T, D>(a), stream, a);
    if (w.rows == 32) ok = launch("bias_forward_kernel", bias_forward_kernel<T, D>, groups, walk_lds<T, D>(a), stream, a);
    if constexpr (BiasStage<T, D>::SUBS == 2)
        if (w.rows == 64) ok = launch("bias_forward_dense_kernel", bias_forward_dense_kernel<T, D, false>, groups, stages_lds<T, D>(a), stream, a);
    if (!ok) return false;
    if (w.splits > 1 && !launch("bias_merge_kernel", bias_merge_kernel<T, D>, nb * a.strips32, 0, stream, a)) return false;
    if (!c.Mean) return true;
    a.splits = room ? mean_splits(c) : 1;
    if (!launch("bias_mean_kernel", bias_mean_kernel<T, D>, strips_of(a.Lq, 64) * strips_of(a.Lk, 64) * a.splits, 0, stream, a)) return false;
    if (a.splits == 1) return true;
    const long long n = (long long)a.Lq * a.Lk;
    hipLaunchKernelGGL(bias_mean_merge_kernel, dim3((unsigned)std::min((n + 255) / 256, 4096LL)), dim3(256), 0, stream, a.part, a.mean, n, a.splits,
                       1.f / nb);
    return check_launch("bias_mean_merge_kernel");
}

template <class T, int D>
static bool backward(const Call& c, hipStream_t stream) {
    BiasCall a = device_call(c);
    const long long nb = (long long)a.B * a.H;
    const Walk row = walk_of(c, a.Lq, a.Lk, true, Pass::ROW), col = walk_of(c, a.Lk, a.Lq, true, Pass::COL);
    a.delta = c.workspace;
    a.tables = a.delta + ((nb * a.Lq + 3) & ~3LL);
    a.part = a.tables + ((nb * col.strips * col.splits * a.buckets + 3) & ~3LL);
    take(a, row, a.Lq);
    const char* name = row.rows > 32 ? "bias_backward_row_dense_kernel" : "bias_backward_row_kernel";
    long long groups = nb * row.strips * row.splits;
    bool ok = true;
    if (row.rows == 128) ok = launch(name, bias_backward_row_dense_kernel<T, D, true>, groups, stages_lds<T, D>(a), stream, a);
    if (row.rows == 32) ok = launch(name, bias_backward_row_kernel<T, D>, groups, walk_lds<T, D>(a), stream, a);
    if constexpr (BiasStage<T, D>::SUBS == 2)
        if (row.rows == 64) ok = launch(name, bias_backward_row_dense_kernel<T, D, false>, groups, stages_lds<T, D>(a), stream, a);
    if (!ok) return false;
    if constexpr (sizeof(T) == 4) {  // (bf16 strips are never cut)
        if (row.splits > 1 && !launch("bias_merge_row_kernel", bias_merge_row_kernel<T, D>, nb * a.strips32, 0, stream, a)) return false;
    }
    take(a, col, a.Lk);
    const size_t hist = HistLds::bytes(a.R);
    name = col.rows > 32 ? "bias_backward_col_dense_kernel" : "bias_backward_col_kernel";
    groups = nb * col.strips * col.splits;
    const size_t staged = stages_lds<T, D>(a) + hist + 2048;
    if (col.rows == 128) ok = launch(name, bias_backward_col_dense_kernel<T, D, true>, groups, staged, stream, a);
    if (col.rows == 32) ok = launch(name, bias_backward_col_kernel<T, D>, groups, walk_lds<T, D>(a) + hist, stream, a);
    if constexpr (BiasStage<T, D>::SUBS == 2)
        if (col.rows == 64) ok = launch(name, bias_backward_col_dense_kernel<T, D, false>, groups, staged, stream, a);
    if (!ok) return false;
    if constexpr (sizeof(T) == 4) {
        if (col.splits > 1 && !launch("bias_merge_col_kernel", bias_merge_col_kernel<T, D>, nb * a.strips32, 0, stream, a)) return false;
    }
    hipLaunchKernelGGL((bias_table_kernel<T>), dim3((unsigned)(a.buckets * a.H)), dim3(256), 0, stream, a, reinterpret_cast<T*>(c.dweight));
    return check_launch("bias_table_kernel");
}

long long bias_workspace(const Call* c, int backward) {
    const char* who = "spion_bias_workspace";
    if (!c) {
        set_error("%s: null pointer", who);
        return -1;
    }
    return sizes_ok(who, *c) ? workspace_floats(*c, backward != 0) : -1;
}

int bias_forward(const Call* c, hipStream_t stream) {
    const char* who = "spion_bias_attention_forward";
    if (!c || !c->weight || !c->buckets || !c->Lse) {
        set_error("%s: null pointer", who);
        return 1;
    }
    if (!sizes_ok(who, *c) || !heads_ok(who, "Q", *c, c->Q, c->q_len, false) || !heads_ok(who, "K", *c, c->K, c->k_len, false) ||
        !heads_ok(who, "V", *c, c->V, c->k_len, false) || !heads_ok(who, "Out", *c, c->Out, c->q_len, true))
        return 1;
    if (c->Mean && c->mat) {
        set_error("%s: the mean map is of the dense phase, without a pattern", who);
        return 1;
    }
    if (reinterpret_cast<uintptr_t>(c->workspace) % 16) {
        set_error("%s: the workspace is not 16-byte aligned", who);
        return 1;
    }
    if (c->Mean && strips_of(c->q_len, 64) * strips_of(c->k_len, 64) > MOST_GROUPS) {
        set_error("%s: mean map too large", who);
        return 1;
    }
    const bool ok = c->bf16 ? (c->head_dim == 32 ? forward<__bf16, 32>(*c, stream) : forward<__bf16, 64>(*c, stream))
                            : (c->head_dim == 32 ? forward<float, 32>(*c, stream) : forward<float, 64>(*c, stream));
    return ok ? 0 : 1;
}

int bias_backward(const Call* c, hipStream_t stream) {
    const char* who = "spion_bias_attention_backward";
    if (!c || !c->weight || !c->dweight || !c->buckets || !c->Lse || !c->workspace) {
        set_error("%s: null pointer", who);
        return 1;
    }
    if (!sizes_ok(who, *c) || !heads_ok(who, "Q", *c, c->Q, c->q_len, false) || !heads_ok(who, "K", *c, c->K, c->k_len, false) ||
        !heads_ok(who, "V", *c, c->V, c->k_len, false) || !heads_ok(who, "Out", *c, c->Out, c->q_len, false) || !heads_ok(who, "dO", *c, c->dO, c->q_len, false) ||
        !heads_ok(who, "dQ", *c, c->dQ, c->q_len, true) || !heads_ok(who, "dK", *c, c->dK, c->k_len, true) || !heads_ok(who, "dV", *c, c->dV, c->k_len, true))
        return 1;
    if (reinterpret_cast<uintptr_t>(c->workspace) % 16) {
        set_error("%s: the workspace is not 16-byte aligned", who);
        return 1;
    }
    if (c->workspace_floats < workspace_floats(*c, true)) {
        set_error("%s: workspace of %lld floats, %lld expected", who, c->workspace_floats, workspace_floats(*c, true));
        return 1;
    }
    const bool ok = c->bf16 ? (c->head_dim == 32 ? backward<__bf16, 32>(*c, stream) : backward<__bf16, 64>(*c, stream))
                            : (c->head_dim == 32 ? backward<float, 32>(*c, stream) : backward<float, 64>(*c, stream));
    return ok ? 0 : 1;
}

}  // namespace spion

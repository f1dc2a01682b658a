// Host side of the attention of queries to keys of another length (kernels: cross_kernels.h): argument checks, launch shapes,
// workspaces.  No handle: sizes come with the call, and nothing is kept from one call for another.
#include "cross_kernels.h"
#include "common.h"
#include "../../include/spion_hip.h"

#include <algorithm>
#include <climits>

namespace spion {

typedef spion_cross_attention Cross;

static long long tiles_of(long long rows, long long tile = 32) { return (rows + tile - 1) / tile; }
static int each_of(const Cross& c) { return c.heads / c.key_heads; }
static long long rows_of(const Cross& c) { return (long long)each_of(c) * c.q_len; }

// Work-groups of 256 threads that a launch holds (2^32 threads and more are refused by the runtime, in the middle of a call).
constexpr long long CROSS_MOST_GROUPS = (1 << 24) - 1;

// How one side of a call is walked: in strips of 128 rows over shared stages, or of 32 with the tiles dealt to the wavefronts, and the
// other side in `splits` pieces.
enum class CrossPass { FORWARD, ROW, COL };
struct CrossWalk {
    int rows;
    int strips, splits, per_split;  // tiles of 32 to a piece
};
// All rows of a group in one strip of 32: the backward is one pass over the keys.
static bool cross_one_strip(const Cross& c) { return rows_of(c) <= 32; }

// Which, by an estimate of the launch's time, us.  A CU's work-groups share it: a launch takes the most work-groups that a CU has, times a piece's
// tiles, times what a tile (strips of 32: four tiles, one to a wavefront) takes, measured with one work-group to a CU in the forward; the row
// pass takes 1.3 times, the column pass 1.75 times that; and where the registers of two fit a CU, several take 0.8 of that (bf16, d = 64: 0.49 us
// a tile of 32 keys and 128 rows alone, 0.41 with four of them; 64 fp32 heads of 16 rows, 4096 padded keys, d = 32, training: 66 us in four pieces
// each, 57 in eight).  All rows in one strip: K and V come from memory
// once, at 20 bytes a ns to a CU.  Pieces cost a second launch, and their sums are written and read at some 4 TB/s.
//   us, forward, one launch / its best cut in strips of 128, strips of 32:  64 heads of 512 x 512, bf16, d = 64: 14 / 22, 17;  32 of 256 x 256: 9 / 14, 7
//   16 of 1024 x 4096: 63 / 37, 41;  d = 128 97 / 60, 93;  fp32 199 / 96, 159;  64 of 256 x 1024, fp32, d = 32: 35 / 25, 23
// At most eight work-groups to a CU where there are pieces, so the workspace is bounded.
static double cross_tile_us(const Cross& c, CrossPass pass, bool few) {
    static const double wide_us[2][3] = {{0.85, 1.5, 3.2}, {0.25, 0.45, 0.75}}, few_us[2][3] = {{1.15, 2.4, 6.}, {0.4, 0.6, 1.35}};
    const int d = c.head_dim == 32 ? 0 : c.head_dim == 64 ? 1 : 2, bf16 = c.bf16 ? 1 : 0;
    const double us = (few ? few_us : wide_us)[bf16][d] * (pass == CrossPass::FORWARD ? 1. : pass == CrossPass::ROW ? 1.3 : 1.75);
    return few && pass != CrossPass::COL && cross_one_strip(c) ? std::max(us, 4 * 64 * c.head_dim * (c.bf16 ? 2 : 4) / 20e3) : us;
}
static CrossWalk cross_walk_of(const Cross& c, CrossPass pass, bool can_split) {
    const long long own = pass == CrossPass::COL ? c.k_len : rows_of(c), other = pass == CrossPass::COL ? rows_of(c) : c.k_len;
    const long long groups = (long long)c.batch * c.key_heads, tiles = tiles_of(other), cus = device_cus();
    const bool must = pass != CrossPass::COL && cross_one_strip(c);
    CrossWalk w{};
    double least = 0;
    for (int few = must; few <= 1; ++few) {
        const int rows = few ? 32 : 128, unit = few ? 1 : 2;
        const long long strips = tiles_of(own, rows), steps = tiles_of(tiles, few ? 4 : unit);
        const double us = cross_tile_us(c, pass, few) * (few ? 1 : unit);
        const bool two = c.bf16 ? !few || c.head_dim < 128 : c.head_dim == 32;  // (two work-groups' registers fit a CU)
        if (groups * strips > CROSS_MOST_GROUPS) continue;  // (strips of 128 are few enough: cross_sizes_ok)
        for (long long n = 1; n == 1 || (can_split && n <= std::min(steps / 2, 64LL) && groups * strips * n <= 8 * cus); ++n) {
            const long long rounds = tiles_of(groups * strips * n, cus), each = tiles_of(steps, n);
            double cost = 3 + rounds * each * us * (rounds > 1 && two ? 0.8 : 1.);
            if (n > 1) cost += 3 + (pass == CrossPass::COL ? 2 : 1) * groups * own * n * c.head_dim * 8 / 4e6;
            if (w.rows && cost >= least) continue;
            least = cost;
            w.rows = rows;
            w.strips = (int)strips;
            w.per_split = (int)(each * (few ? 4 : unit));
            w.splits = few ? (int)n : (int)tiles_of(steps, each);  // none of them empty
        }
    }
    return w;
}

static long long cross_floats(const Cross& c, bool backward) {
    const long long groups = (long long)c.batch * c.key_heads, rows = rows_of(c);
    if (!backward) {
        const CrossWalk w = cross_walk_of(c, CrossPass::FORWARD, true);
        return w.splits > 1 ? groups * tiles_of(rows) * w.splits * (32 * c.head_dim + 64) : 0;
    }
    const CrossWalk row = cross_walk_of(c, CrossPass::ROW, true), col = cross_walk_of(c, CrossPass::COL, true);
    const long long a = row.splits > 1 ? groups * tiles_of(rows) * row.splits * 32 * c.head_dim : 0;
    const long long b = !cross_one_strip(c) && col.splits > 1 ? groups * tiles_of(c.k_len) * col.splits * 64 * c.head_dim : 0;
    return ((groups * rows + 3) & ~3LL) + std::max(a, b);  // D, rounded up to whole pieces of 16 bytes, and the pieces
}

static bool cross_sizes_ok(const char* who, const Cross& c) {
    if (c.batch < 1 || c.heads < 1 || c.key_heads < 1 || c.q_len < 1 || c.k_len < 1) {
        set_error("%s: sizes are positive", who);
        return false;
    }
    if (c.heads % c.key_heads) {
        set_error("%s: %d heads over %d heads of keys: a multiple expected", who, c.heads, c.key_heads);
        return false;
    }
    if (c.head_dim != 32 && c.head_dim != 64 && c.head_dim != 128) {
        set_error("%s: head_dim %d, 32, 64 or 128 expected", who, c.head_dim);
        return false;
    }
    if (rows_of(c) > (1 << 29) || c.k_len > (1 << 29)) {
        set_error("%s: up to 2^29 keys, and rows of the heads that share them", who);
        return false;
    }
    const long long groups = (long long)c.batch * c.key_heads;
    if (groups > CROSS_MOST_GROUPS || groups * tiles_of(std::max<long long>(rows_of(c), c.k_len), 128) > CROSS_MOST_GROUPS) {
        set_error("%s: too many heads and rows for one launch: 2^24 strips of 128 rows, or of 128 keys", who);
        return false;
    }
    if (c.key_mask && c.mask_bytes != 1 && c.mask_bytes != 4) {
        set_error("%s: a key mask has 1 or 4 bytes a key", who);
        return false;
    }
    return true;
}

// heads: of those that one work-group reads (a group of queries, a head of keys), `rows` rows each
static bool cross_heads_ok(const char* who, const char* name, const Cross& c, const spion_heads& t, int heads, int rows, bool written) {
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
    constexpr long long most = INT_MAX;
    if (t.row_stride > (1 << 24) / e || (heads > 1 && t.head_stride > most / e) ||
        (heads - 1) * t.head_stride * e > most || (heads - 1) * t.head_stride * e + (rows - 1) * t.row_stride * e + c.head_dim * e > most) {
        set_error("%s: %s: rows up to 2^24 bytes apart and heads of a group within 2^31 bytes expected", who, name);
        return false;
    }
    return true;
}
static bool cross_queries_ok(const char* who, const char* name, const Cross& c, const spion_heads& t, bool written) {
    return cross_heads_ok(who, name, c, t, each_of(c), c.q_len, written);
}
static bool cross_keys_ok(const char* who, const char* name, const Cross& c, const spion_heads& t, bool written) {
    return cross_heads_ok(who, name, c, t, 1, c.k_len, written);
}

static CrossCall cross_device_call(const Cross& c) {
    const auto at = [&](const spion_heads& t) {
        const int e = c.bf16 ? 2 : 4;
        return HeadsAt{reinterpret_cast<const char*>(t.p), t.batch_stride * e, t.head_stride * e, t.row_stride * e};
    };
    CrossCall a{};
    a.q = at(c.Q), a.k = at(c.K), a.v = at(c.V), a.o = at(c.Out);
    a.dout = at(c.dO), a.dq = at(c.dQ), a.dk = at(c.dK), a.dv = at(c.dV);
    a.mask = c.key_mask, a.mask_bytes = c.mask_bytes, a.lse = c.Lse;
    a.B = c.batch, a.G = c.key_heads, a.each = each_of(c), a.Lq = c.q_len, a.Lk = c.k_len, a.rows = (int)rows_of(c);
    // ceil(2^(31 + l) / Lq) with 2^(l - 1) < Lq <= 2^l: its error times r < 2^31 stays below 2^(31 + l), so r / Lq comes out whole
    int l = 0;
    while ((1LL << l) < a.Lq) ++l;
    a.magic = (unsigned)(((1ULL << (31 + l)) + a.Lq - 1) / a.Lq);
    a.shift = 31 + l;
    a.scale = 1.0f / sqrtf((float)c.head_dim);
    return a;
}
static void cross_take(CrossCall& a, const CrossWalk& w) {
    a.strips = w.strips;
    a.splits = w.splits;
    a.per_split = w.per_split;
}

template <class K>
static bool cross_launch(const char* name, K kernel, long long groups, size_t lds, hipStream_t stream, const CrossCall& a) {
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

template <int D, class K>
static bool cross_join(const char* name, K few, K many, long long groups, long long rows, hipStream_t stream, const CrossCall& a) {
    if (a.splits > 8) return cross_launch(name, many, groups * rows, 0, stream, a);
    return cross_launch(name, few, groups * tiles_of(rows, CrossJoin<D, false>::ROWS), 0, stream, a);
}

template <class T, int D>
struct CrossRun {
    static constexpr size_t STAGES = cross_stages_bytes<T, D>() + sizeof(CrossLds);
    static bool forward(const Cross& c, hipStream_t stream) {
        CrossCall a = cross_device_call(c);
        const long long groups = (long long)a.B * a.G;
        const CrossWalk w = cross_walk_of(c, CrossPass::FORWARD, c.workspace && c.workspace_floats >= cross_floats(c, false));
        cross_take(a, w);
        a.part = c.workspace;
        const long long n = groups * w.strips * w.splits;
        bool ok = false;
        if (w.rows == 128) ok = cross_launch("cross_forward_kernel", cross_forward_kernel<T, D>, n, STAGES, stream, a);
        if (w.rows == 32) ok = cross_launch("cross_forward_few_kernel", cross_forward_few_kernel<T, D>, n, cross_tiles_bytes<T, D>(), stream, a);
        return ok && (w.splits == 1 || cross_join<D>("cross_merge_kernel", cross_merge_kernel<T, D, false>, cross_merge_kernel<T, D, true>, groups, a.rows, stream, a));
    }
    static bool backward(const Cross& c, hipStream_t stream) {
        constexpr bool BF16 = sizeof(T) == 2;
        // dS in two bf16 numbers up to 256 keys, where the rounding of O in D shows (128 heads of 1024 x 256: d = 64 81 us, and 77 without; d = 128 137 and
        // 128; of 512, where it shows no more, 121 and 109).  By the keys there are: the host does not know how many a mask leaves.  dV has no D in it
        // and takes P in one number.
        const bool fine = BF16 && c.k_len <= 256;
        CrossCall a = cross_device_call(c);
        const long long groups = (long long)a.B * a.G;
        const CrossWalk row = cross_walk_of(c, CrossPass::ROW, true), col = cross_walk_of(c, CrossPass::COL, true);
        a.delta = c.workspace;
        a.part = a.delta + ((groups * a.rows + 3) & ~3LL);
        cross_take(a, row);
        long long n = groups * row.strips * row.splits;
        bool ok = false;
        if (row.rows == 128) ok = cross_launch("cross_backward_row_kernel", fine ? cross_backward_row_kernel<T, D, BF16> : cross_backward_row_kernel<T, D, false>, n, STAGES, stream, a);
        if (cross_one_strip(c)) ok = cross_launch("cross_backward_few_kernel", cross_backward_few_kernel<T, D>, n, cross_few_bytes<T, D>(), stream, a);
        else if (row.rows == 32)
            ok = cross_launch("cross_backward_row_few_kernel", cross_backward_row_few_kernel<T, D>, n, cross_tiles_bytes<T, D>() + cross_shared_bytes<T, D>(), stream, a);
        if (!ok) return false;
        if (row.splits > 1 &&
            !cross_join<D>("cross_merge_row_kernel", cross_merge_row_kernel<T, D, false>, cross_merge_row_kernel<T, D, true>, groups, a.rows, stream, a))
            return false;
        if (cross_one_strip(c)) return true;  // (with all three gradients)
        cross_take(a, col);
        n = groups * col.strips * col.splits;
        if (col.rows == 128)
            ok = cross_launch("cross_backward_col_kernel", fine ? cross_backward_col_kernel<T, D, BF16> : cross_backward_col_kernel<T, D, false>, n, STAGES + 1024, stream, a);
        if (col.rows == 32)
            ok = cross_launch("cross_backward_col_few_kernel", cross_backward_col_few_kernel<T, D>, n, cross_col_few_bytes<T, D>(), stream, a);
        if (!ok) return false;
        return col.splits == 1 ||
               cross_join<D>("cross_merge_col_kernel", cross_merge_col_kernel<T, D, false>, cross_merge_col_kernel<T, D, true>, groups, a.Lk, stream, a);
    }
};

template <class T>
static bool cross_run(const Cross& c, bool backward, hipStream_t stream) {
    switch (c.head_dim) {
        case 32: return backward ? CrossRun<T, 32>::backward(c, stream) : CrossRun<T, 32>::forward(c, stream);
        case 64: return backward ? CrossRun<T, 64>::backward(c, stream) : CrossRun<T, 64>::forward(c, stream);
        default: return backward ? CrossRun<T, 128>::backward(c, stream) : CrossRun<T, 128>::forward(c, stream);
    }
}

long long cross_workspace(const Cross* c, int backward) {
    const char* who = "spion_cross_workspace";
    if (!c) {
        set_error("%s: null pointer", who);
        return -1;
    }
    return cross_sizes_ok(who, *c) ? cross_floats(*c, backward != 0) : -1;
}

int cross_forward(const Cross* c, hipStream_t stream) {
    const char* who = "spion_cross_attention_forward";
    if (!c || !c->Lse) {
        set_error("%s: null pointer", who);
        return 1;
    }
    if (!cross_sizes_ok(who, *c) || !cross_queries_ok(who, "Q", *c, c->Q, false) || !cross_keys_ok(who, "K", *c, c->K, false) ||
        !cross_keys_ok(who, "V", *c, c->V, false) || !cross_queries_ok(who, "Out", *c, c->Out, true))
        return 1;
    if (reinterpret_cast<uintptr_t>(c->workspace) % 16) {
        set_error("%s: the workspace is not 16-byte aligned", who);
        return 1;
    }
    return (c->bf16 ? cross_run<__bf16>(*c, false, stream) : cross_run<float>(*c, false, stream)) ? 0 : 1;
}

int cross_backward(const Cross* c, hipStream_t stream) {
    const char* who = "spion_cross_attention_backward";
    if (!c || !c->Lse || !c->workspace) {
        set_error("%s: null pointer", who);
        return 1;
    }
    if (!cross_sizes_ok(who, *c) || !cross_queries_ok(who, "Q", *c, c->Q, false) || !cross_keys_ok(who, "K", *c, c->K, false) ||
        !cross_keys_ok(who, "V", *c, c->V, false) || !cross_queries_ok(who, "Out", *c, c->Out, false) ||
        !cross_queries_ok(who, "dO", *c, c->dO, false) || !cross_queries_ok(who, "dQ", *c, c->dQ, true) ||
        !cross_keys_ok(who, "dK", *c, c->dK, true) || !cross_keys_ok(who, "dV", *c, c->dV, true))
        return 1;
    if (reinterpret_cast<uintptr_t>(c->workspace) % 16) {
        set_error("%s: the workspace is not 16-byte aligned", who);
        return 1;
    }
    if (c->workspace_floats < cross_floats(*c, true)) {
        set_error("%s: workspace of %lld floats, %lld expected", who, c->workspace_floats, cross_floats(*c, true));
        return 1;
    }
    return (c->bf16 ? cross_run<__bf16>(*c, true, stream) : cross_run<float>(*c, true, stream)) ? 0 : 1;
}

}  // namespace spion

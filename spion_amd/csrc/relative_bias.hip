// Host side of the attention with a learned bias by buckets of relative position (kernels: bias_kernels.h): argument checks,
// launch shapes, workspaces.  No handle: sizes come with the call, and nothing is kept from one call for another.
#include "bias_dense_kernels.h"
#include "common.h"
#include "../../include/spion_hip.h"

#include <algorithm>
#include <climits>

namespace spion {

typedef spion_bias_attention Call;

static long long strips_of(int rows) { return (rows + 31) / 32; }

// Pieces of the keys a forward strip is walked in.  Launches with fewer work-groups than twice the machine's CUs are split
// until they have that many, each wavefront keeping at least two tiles.
static int forward_splits(const Call& c) {
    const long long groups = (long long)c.batch * c.heads * strips_of(c.q_len), tiles = strips_of(c.k_len);
    const long long want = (2LL * device_cus() + groups - 1) / groups, most = tiles / 8;
    return (int)std::max(1LL, std::min({want, most, 64LL}));
}

static long long workspace_floats(const Call& c, bool backward) {
    const long long nb = (long long)c.batch * c.heads;
    if (backward) return nb * c.q_len + nb * strips_of(c.k_len) * c.num_buckets;
    const int s = forward_splits(c);
    return s > 1 ? nb * strips_of(c.q_len) * s * (32 * c.head_dim + 96) : 0;
}

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
    if ((long long)c.batch * c.heads > INT_MAX / 64 || (long long)c.batch * c.heads * strips_of((int)longest) > INT_MAX / 64) {
        set_error("%s: too many heads and rows for one launch", who);
        return false;
    }
    if (c.mat && (c.block_size < 32 || c.block_size % 32 || c.q_len != c.k_len || c.offset != 0)) {
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

static bool heads_ok(const char* who, const char* name, const Call& c, const spion_heads& t, bool written) {
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

// Whether a side of `rows` rows is walked in strips of 128: without a pattern, and with strips enough for the machine.
static bool dense_strips(const Call& c, int rows) {
    return !c.mat && (long long)c.batch * c.heads * ((rows + 127) / 128) >= 2 * device_cus();
}
template <class T, int D>
static size_t stages_lds(const BiasCall& a) {
    return bias_stages_bytes<T, D>() + bias_floats(a.R) * 4 + sizeof(ScanLds);
}

template <class T, int D>
static size_t walk_lds(const BiasCall& a) {
    return bias_tiles_bytes<T, D>() + bias_floats(a.R) * 4 + sizeof(ScanLds);
}

template <class T, int D>
static bool mean_map(const Call& c, const BiasCall& a, hipStream_t stream) {
    return !c.Mean || launch("bias_mean_kernel", bias_mean_kernel<T, D>, strips_of(a.Lq) * strips_of(a.Lk), 0, stream, a);
}

template <class T, int D>
static bool forward(const Call& c, hipStream_t stream) {
    BiasCall a = device_call(c);
    const long long nb = (long long)a.B * a.H, tiles = strips_of(a.Lk);
    if (dense_strips(c, a.Lq)) {
        a.strips = (a.Lq + 127) / 128;
        return launch("bias_forward_dense_kernel", bias_forward_dense_kernel<T, D>, nb * a.strips, stages_lds<T, D>(a), stream, a) && mean_map<T, D>(c, a, stream);
    }
    a.strips = (int)strips_of(a.Lq);
    a.splits = forward_splits(c);
    if (a.splits > 1 && (!c.workspace || c.workspace_floats < workspace_floats(c, false))) a.splits = 1;
    a.per_split = (int)((tiles + a.splits - 1) / a.splits);
    a.splits = (int)((tiles + a.per_split - 1) / a.per_split);  // none of them empty
    a.part = c.workspace;
    if (!launch("bias_forward_kernel", bias_forward_kernel<T, D>, nb * a.strips * a.splits, walk_lds<T, D>(a), stream, a)) return false;
    if (a.splits > 1 && !launch("bias_merge_kernel", bias_merge_kernel<T, D>, nb * a.strips, 0, stream, a)) return false;
    return mean_map<T, D>(c, a, stream);
}

template <class T, int D>
static bool backward(const Call& c, hipStream_t stream) {
    BiasCall a = device_call(c);
    const long long nb = (long long)a.B * a.H;
    a.delta = c.workspace;
    a.part = c.workspace + nb * a.Lq;
    const bool rows = dense_strips(c, a.Lq), cols = dense_strips(c, a.Lk);
    a.strips = rows ? (a.Lq + 127) / 128 : (int)strips_of(a.Lq);
    if (!(rows ? launch("bias_backward_row_dense_kernel", bias_backward_row_dense_kernel<T, D>, nb * a.strips, stages_lds<T, D>(a), stream, a)
               : launch("bias_backward_row_kernel", bias_backward_row_kernel<T, D>, nb * a.strips, walk_lds<T, D>(a), stream, a)))
        return false;
    a.strips = cols ? (a.Lk + 127) / 128 : (int)strips_of(a.Lk);
    const size_t hist = HistLds::bytes(a.R);
    if (!(cols ? launch("bias_backward_col_dense_kernel", bias_backward_col_dense_kernel<T, D>, nb * a.strips, stages_lds<T, D>(a) + hist + 2048, stream, a)
               : launch("bias_backward_col_kernel", bias_backward_col_kernel<T, D>, nb * a.strips, walk_lds<T, D>(a) + hist, stream, a)))
        return false;
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
    if (!sizes_ok(who, *c) || !heads_ok(who, "Q", *c, c->Q, false) || !heads_ok(who, "K", *c, c->K, false) ||
        !heads_ok(who, "V", *c, c->V, false) || !heads_ok(who, "Out", *c, c->Out, true))
        return 1;
    if (c->Mean && c->mat) {
        set_error("%s: the mean map is of the dense phase, without a pattern", who);
        return 1;
    }
    if (c->Mean && strips_of(c->q_len) * strips_of(c->k_len) > INT_MAX) {
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
    if (!sizes_ok(who, *c) || !heads_ok(who, "Q", *c, c->Q, false) || !heads_ok(who, "K", *c, c->K, false) ||
        !heads_ok(who, "V", *c, c->V, false) || !heads_ok(who, "Out", *c, c->Out, false) || !heads_ok(who, "dO", *c, c->dO, false) ||
        !heads_ok(who, "dQ", *c, c->dQ, true) || !heads_ok(who, "dK", *c, c->dK, true) || !heads_ok(who, "dV", *c, c->dV, true))
        return 1;
    if (c->workspace_floats < workspace_floats(*c, true)) {
        set_error("%s: workspace of %lld floats, %lld expected", who, c->workspace_floats, workspace_floats(*c, true));
        return 1;
    }
    if ((long long)c->num_buckets * c->heads > INT_MAX) {
        set_error("%s: table too large", who);
        return 1;
    }
    const bool ok = c->bf16 ? (c->head_dim == 32 ? backward<__bf16, 32>(*c, stream) : backward<__bf16, 64>(*c, stream))
                            : (c->head_dim == 32 ? backward<float, 32>(*c, stream) : backward<float, 64>(*c, stream));
    return ok ? 0 : 1;
}

}  // namespace spion

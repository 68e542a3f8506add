// C ABI of the row matching operators and the patch descriptors (include/custma.h): checks, choice of
// variants and splits, workspace.  As in capi.hip nothing is allocated, nothing waits for the device, and
// every launch goes to the caller's stream.
#include <stdio.h>

#include "match_launch.h"

using namespace custma;

namespace {
constexpr int64_t kMaxLen = (int64_t)1 << 30;
constexpr int64_t kMaxStride = (int64_t)1 << 24;
constexpr int64_t kMaxRows = (int64_t)1 << 46;
constexpr int kMaxWide = 16384;
constexpr int64_t kMaxBlocks = ((int64_t)1 << 24) - 1;  // a launch counts its threads in 32 bits

template <typename... A>
int refuse(int code, const char* fmt, A... args) {
    char text[320];
    if constexpr (sizeof...(args) > 0) snprintf(text, sizeof(text), fmt, args...);
    else snprintf(text, sizeof(text), "%s", fmt);
    return capi_fail(code, text);
}
int ran(hipError_t e, const char* what) {
    if (e == hipSuccess) return CUSTMA_OK;
    return refuse(CUSTMA_E_LAUNCH, "%s: HIP error %d (%s)", what, (int)e, hipGetErrorString(e));
}
size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

int64_t at_most(int64_t v, int64_t top) { return v < top ? v : top; }

int make_match(const custma_match_geo* c, int32_t op, MatchGeo* g) {
    if (!c) return refuse(CUSTMA_E_NULL, "null geometry");
    if (op < CUSTMA_MATCH_ATTENTION || op > CUSTMA_MATCH_ENTROPY_BACKWARD) return refuse(CUSTMA_E_ARG, "unknown operation %d", op);
    const bool entropy = op >= CUSTMA_MATCH_ENTROPY;
    if (c->dtype != CUSTMA_F16 && c->dtype != CUSTMA_BF16)
        return refuse(CUSTMA_E_ARG, "unsupported dtype code %d (float16=1, bfloat16=2)", c->dtype);
    if (c->batch < 0 || c->query_len < 0 || c->key_len < 0 || c->batch >= kMaxLen || c->query_len >= kMaxLen || c->key_len >= kMaxLen)
        return refuse(CUSTMA_E_ARG, "sizes must be in [0, 2^30), got batch=%lld query_len=%lld key_len=%lld",
                      (long long)c->batch, (long long)c->query_len, (long long)c->key_len);
    if (c->kv_heads < 1 || c->group < 1 || c->query_len * c->group >= kMaxLen)
        return refuse(CUSTMA_E_ARG, "kv_heads and group must be at least 1 and query_len * group below 2^30");
    // so that no size computed from them leaves 64 bits
    const unsigned __int128 rows = (unsigned __int128)c->batch * c->query_len * ((uint64_t)c->kv_heads * c->group);
    if (rows >= kMaxRows || (unsigned __int128)c->batch * c->key_len * c->kv_heads >= kMaxRows)
        return refuse(CUSTMA_E_UNSUPPORTED, "batch * length * heads must be below 2^46");
    const bool wide = entropy && c->channels > kMatchMaxC;
    if (c->channels < 8 || c->channels % 8 || c->channels > (entropy ? kMaxWide : kMatchMaxC))
        return refuse(CUSTMA_E_ARG, "channels must be a multiple of 8 in [8, %d], got %d", entropy ? kMaxWide : kMatchMaxC, c->channels);
    if (entropy ? c->value_channels != 0 : (c->value_channels < 8 || c->value_channels % 8 || c->value_channels > kMatchMaxC))
        return refuse(CUSTMA_E_ARG, "value_channels must be a multiple of 8 in [8, %d] (0 for the cross entropy), got %d", kMatchMaxC, c->value_channels);
    if (!(c->scale - c->scale == 0.f)) return refuse(CUSTMA_E_ARG, "scale must be finite");
    if (c->left < -1 || c->right < -1 || c->sinks < 0)
        return refuse(CUSTMA_E_ARG, "left and right must be at least 0 (or -1), sinks at least 0");
    if (entropy && (c->kv_heads != 1 || c->group != 1 || c->sinks || c->offset || c->length))
        return refuse(CUSTMA_E_ARG, "the cross entropy takes no heads, sinks, offsets or lengths");
    if (wide && (c->left >= 0 || c->right >= 0))
        return refuse(CUSTMA_E_UNSUPPORTED, "a window needs at most %d channels, got %d", kMatchMaxC, c->channels);
    for (int i = 0; i < 3; ++i)
        if (c->q_stride[i] % 8 || c->k_stride[i] % 8 || (!entropy && c->v_stride[i] % 8) || c->q_stride[i] < 0 ||
            c->k_stride[i] < 0 || (!entropy && c->v_stride[i] < 0))
            return refuse(CUSTMA_E_ARG, "strides must be non-negative multiples of 8 elements");
    // a tile's rows are addressed in 32 bits from its first one: key tiles always, tiles of query rows and of the output's
    // gradient in the gradients of the keys
    const bool back = op == CUSTMA_MATCH_ATTENTION_BACKWARD || op == CUSTMA_MATCH_ENTROPY_BACKWARD;
    if (c->k_stride[1] >= kMaxStride || (!entropy && c->v_stride[1] >= kMaxStride) ||
        (back && (c->q_stride[1] >= kMaxStride || (c->group > 1 && c->q_stride[2] >= kMaxStride))))
        return refuse(CUSTMA_E_UNSUPPORTED, "position strides (and for gradients query head strides) must be below 2^24 elements");
    if (back && !entropy && (int64_t)c->kv_heads * c->group >= kMaxStride / c->value_channels)
        return refuse(CUSTMA_E_UNSUPPORTED, "gradients need heads * value_channels below 2^24");
    for (int i = 0; i < 3; ++i) {
        g->qs[i] = c->q_stride[i];
        g->ks[i] = c->k_stride[i];
        g->vs[i] = entropy ? 0 : c->v_stride[i];
    }
    g->offset = c->offset;
    g->length = c->length;
    g->B = (int32_t)c->batch;
    g->Lq = (int32_t)c->query_len;
    g->Lk = (int32_t)c->key_len;
    g->Hkv = c->kv_heads;
    g->G = c->group;
    g->C = c->channels;
    g->Cv = c->value_channels;
    g->left = c->left < 0 ? -1 : (int32_t)at_most(c->left, INT32_MAX);
    g->right = c->right < 0 ? -1 : (int32_t)at_most(c->right, INT32_MAX);
    g->sinks = g->left < 0 ? 0 : (int32_t)at_most(c->sinks, c->key_len);
    g->scale = c->scale;
    return CUSTMA_OK;
}

struct Dims {
    int64_t rows;   // B * Lq * heads
    int64_t keys;   // B * Lk * Hkv
};
Dims dims(const MatchGeo& g) { return {(int64_t)g.B * g.Lq * g.heads(), (int64_t)g.B * g.Lk * g.Hkv}; }

// template widths: C in 32, 64, 128, 256; values in 32 or the same width (the larger of the two where they differ)
void widths(const MatchGeo& g, int* hd, int* hdv) {
    const int c = pad_channels(g.C), v = g.Cv ? pad_channels(g.Cv) : 0;
    *hd = v > c ? v : c;
    *hdv = v == 0 ? 0 : v == 32 ? 32 : *hd;
}

// how many keys one query tile can reach, at most
int64_t reach(const MatchGeo& g, int tile_positions) {
    if (g.left < 0 || g.right < 0) return g.Lk;
    return at_most((int64_t)g.left + g.right + tile_positions + g.sinks, g.Lk);
}

// Few rows: the waves of a workgroup split the keys (a tile of 32 rows instead of 128), and where the grid
// would still leave compute units idle the key range is split over workgroups.
struct FwdPlan {
    bool few;
    int nsplit;
};
FwdPlan plan_fwd(const MatchGeo& g) {
    int hd, hdv;
    widths(g, &hd, &hdv);
    FwdPlan p;
    const int few_rows = hd == 256 ? 64 : 32;
    p.few = g.rows() <= few_rows;
    const int br = p.few ? few_rows : 128;
    const int kt = p.few ? (hd == 256 ? 64 : 128) : (hd == 256 ? 32 : 64);
    const int64_t base = cdiv(g.rows(), br) * g.Hkv * g.B;
    const int64_t tiles = cdiv(reach(g, (int)cdiv(br, g.G) + 1), kt);
    int64_t s = base >= 256 || base == 0 ? 1 : cdiv(256, base);
    if (s > tiles) s = tiles;
    p.nsplit = (int)(s < 1 ? 1 : s > 64 ? 64 : s);
    return p;
}

// Key gradients walk the query rows; split them where the grid leaves compute units idle.
int plan_bwd_k(const MatchGeo& g) {
    int hd, hdv;
    widths(g, &hd, &hdv);
    const int64_t base = cdiv(g.Lk, 128) * g.Hkv * g.B;
    const int rt = hd == 256 ? 32 : 64;
    int64_t span = g.Lq;
    if (g.left >= 0 && g.right >= 0) span = at_most((int64_t)g.left + g.right + 128, g.Lq);
    const int64_t tiles = cdiv(span * g.G, rt);
    int64_t s = base >= 256 || base == 0 ? 1 : cdiv(256, base);
    if (s > tiles / 2) s = tiles / 2;
    return (int)(s < 1 ? 1 : s > 32 ? 32 : s);
}
int plan_sinks(const MatchGeo& g) {
    int hd, hdv;
    widths(g, &hd, &hdv);
    const int64_t base = cdiv(g.sinks, 128) * g.Hkv * g.B;
    const int64_t tiles = cdiv((int64_t)g.rows(), hd == 256 ? 32 : 64);
    int64_t s = base == 0 ? 1 : cdiv(512, base);
    if (s > tiles / 2) s = tiles / 2;
    return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

// Workspace, carved in order; with base null it only counts.
struct Carve {
    char* base;
    size_t at = 0;
    template <typename T>
    T* take(size_t n) {
        T* p = base ? (T*)(base + at) : nullptr;
        at += up256(n * sizeof(T));
        return p;
    }
};
struct BwdSpace {
    float *start, *second;
    int32_t* hot;
    float *partials, *scale, *part_k, *part_v, *sink_k, *sink_v, *init_k, *init_v;
    char* go16;
};
void carve_bwd(const MatchGeo& g, bool go32, Carve& c, BwdSpace* w) {
    const Dims d = dims(g);
    const int S = plan_bwd_k(g);
    w->start = c.take<float>(d.rows);
    w->second = c.take<float>(d.rows);
    w->hot = g.Cv ? nullptr : c.take<int32_t>(d.rows);
    w->go16 = go32 ? c.take<char>((size_t)d.rows * g.Cv * 2) : nullptr;
    w->partials = go32 ? c.take<float>(1024) : nullptr;
    w->scale = go32 ? c.take<float>(1) : nullptr;
    w->part_k = S > 1 ? c.take<float>((size_t)S * d.keys * g.C) : nullptr;
    w->part_v = S > 1 && g.Cv ? c.take<float>((size_t)S * d.keys * g.Cv) : nullptr;
    w->sink_k = w->sink_v = w->init_k = w->init_v = nullptr;
    if (g.sinks > 0) {
        const size_t n = (size_t)g.B * g.sinks * g.Hkv;
        const int T = plan_sinks(g);
        w->sink_k = c.take<float>(T * n * g.C);
        w->sink_v = c.take<float>(T * n * g.Cv);
        w->init_k = c.take<float>(n * g.C);
        w->init_v = c.take<float>(n * g.Cv);
    }
}
struct WeightSpace {
    float *weight, *partials, *scale;
};
WeightSpace carve_weights(const MatchGeo& g, Carve& c) {
    return {c.take<float>(dims(g).rows), c.take<float>(1024), c.take<float>(1)};
}
struct FwdSpace {
    float *part, *part_ml;
    double* partials;
};
void carve_fwd(const MatchGeo& g, bool entropy, Carve& c, FwdSpace* w) {
    const Dims d = dims(g);
    if (entropy && g.C > kMatchMaxC) {
        w->part = nullptr;
        w->part_ml = c.take<float>((size_t)2 * wide_splits(g) * d.rows * 4);
    } else {
        const int S = plan_fwd(g).nsplit;
        w->part = S > 1 && !entropy ? c.take<float>((size_t)S * d.rows * g.Cv) : nullptr;
        w->part_ml = S > 1 ? c.take<float>((size_t)S * d.rows * 4) : nullptr;
    }
    w->partials = entropy ? c.take<double>(2 * 1024) : nullptr;
}
size_t need(const custma_match_geo* geo, const MatchGeo& g, int32_t op) {
    Carve c{nullptr};
    if (g.B == 0) return 256;
    if (op == CUSTMA_MATCH_ATTENTION || op == CUSTMA_MATCH_ENTROPY) {
        FwdSpace w;
        if (g.Lq > 0) carve_fwd(g, op == CUSTMA_MATCH_ENTROPY, c, &w);
        return c.at + (op == CUSTMA_MATCH_ENTROPY && g.Lq == 0 ? up256(2 * 1024 * sizeof(double)) : 0) + 256;
    }
    if (op == CUSTMA_MATCH_ENTROPY_BACKWARD) (void)carve_weights(g, c);
    if (op == CUSTMA_MATCH_ENTROPY_BACKWARD && g.C > kMatchMaxC) return c.at + wide_bwd_bytes(g) + 256;
    BwdSpace w;
    carve_bwd(g, op == CUSTMA_MATCH_ATTENTION_BACKWARD && geo->out_f32, c, &w);
    return c.at + 256;
}
int check_space(const custma_match_geo* geo, const MatchGeo& g, int32_t op, const void* ws, size_t bytes) {
    const size_t n = need(geo, g, op);
    if (!ws) return refuse(CUSTMA_E_NULL, "null workspace");
    if (bytes < n) return refuse(CUSTMA_E_WORKSPACE, "workspace too small (%zu < %zu)", bytes, n);
    if ((uintptr_t)ws % 256) return refuse(CUSTMA_E_ARG, "workspace must be 256-byte aligned");
    return CUSTMA_OK;
}
bool unaligned(const void* p) { return (uintptr_t)p % 16 != 0; }
int check_blocks(int64_t blocks) {
    if (blocks > kMaxBlocks) return refuse(CUSTMA_E_UNSUPPORTED, "too many rows for one call (%lld workgroups)", (long long)blocks);
    return CUSTMA_OK;
}
// every launch of a call: tiles of rows, of keys, and the per-row passes
int check_grid(const MatchGeo& g) {
    const Dims d = dims(g);
    int rc = check_blocks(cdiv(g.rows(), 32) * g.Hkv * (int64_t)g.B);
    if (rc || (rc = check_blocks(cdiv(g.Lk, 128) * g.Hkv * (int64_t)g.B))) return rc;
    return check_blocks(cdiv(d.rows * (g.Cv ? (g.Cv + 3) / 4 : 1), 256));
}

#define CUSTMA_BY_HD(fn, ...)                                                              \
    (hd == 32 ? fn##_32(__VA_ARGS__) : hd == 64 ? fn##_64(__VA_ARGS__)                       \
     : hd == 128 ? fn##_128(__VA_ARGS__) : fn##_256(__VA_ARGS__))

hipError_t run_fwd(const MatchGeo& g, int dtype, bool wide_out, const void* q, const void* k, const void* v,
                   const FwdOut& o, hipStream_t s) {
    int hd, hdv;
    widths(g, &hd, &hdv);
    const FwdPlan p = plan_fwd(g);
    hipError_t e = CUSTMA_BY_HD(launch_match_fwd, g, dtype, wide_out, p.few, hdv, q, k, v, o, p.nsplit, s);
    if (e == hipSuccess && p.nsplit > 1) e = launch_match_join(g, dtype, wide_out, o, p.nsplit, s);
    return e;
}

// out (attention): the forward's output, with low; null for the cross entropy
hipError_t run_bwd(const MatchGeo& g, int dtype, BwdArgs a, const BwdSpace& w, const float* lse, const void* out,
                   bool out_f32, const void* low, hipStream_t s) {
    int hd, hdv;
    widths(g, &hd, &hdv);
    hipError_t e = hipSuccess;
    a.start = w.start, a.second = w.second, a.hot = w.hot;
    if (g.Lq > 0) e = launch_match_rows(g, dtype, a, lse, out, out_f32, low, s);
    if (e != hipSuccess) return e;
    if (a.gq && g.Lq > 0) e = CUSTMA_BY_HD(launch_match_bwd_q, g, dtype, hdv, a, s);
    if (e != hipSuccess || (!a.gk && !a.gv) || g.Lk == 0) return e;
    const Dims d = dims(g);
    if (g.sinks > 0) {
        const int T = plan_sinks(g);
        const int64_t n = (int64_t)g.B * g.sinks * g.Hkv;
        BwdArgs b = a;
        b.part_k = w.sink_k;
        b.part_v = a.gv ? w.sink_v : nullptr;
        e = CUSTMA_BY_HD(launch_match_bwd_k, g, dtype, hdv, b, true, T, s);
        if (e == hipSuccess)
            e = launch_match_sum(w.sink_k, T, n * g.C, dtype, true, nullptr, 1.f, w.init_k, w.sink_v, n * g.Cv, 1.f,
                                 a.gv ? w.init_v : nullptr, s);
        if (e != hipSuccess) return e;
        a.init_k = w.init_k;
        a.init_v = w.init_v;
        a.init_keys = g.sinks;
    }
    const int S = plan_bwd_k(g);
    const float lift = hdv ? 1.f : dtype == CUSTMA_F16 ? ldexpf(1.f, -(int)Half16<_Float16>::kLift) : 1.f;
    if (S > 1) {
        a.part_k = w.part_k;
        a.part_v = a.gv ? w.part_v : nullptr;
    }
    e = CUSTMA_BY_HD(launch_match_bwd_k, g, dtype, hdv, a, false, S, s);
    if (S > 1 && e == hipSuccess)
        e = launch_match_sum(w.part_k, S, d.keys * g.C, dtype, false, a.factor, g.scale * lift, a.gk, w.part_v,
                             d.keys * g.Cv, 1.f, a.gv, s);
    return e;
}
}  // namespace

extern "C" {

size_t custma_match_workspace_bytes(const custma_match_geo* geo, int32_t op) {
    MatchGeo g;
    return make_match(geo, op, &g) ? 0 : need(geo, g, op);
}

int custma_match_attention(const custma_match_geo* geo, const void* q, const void* k, const void* v, void* out,
                           void* low, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    MatchGeo g;
    int rc = make_match(geo, CUSTMA_MATCH_ATTENTION, &g);
    if (rc) return rc;
    if (g.B == 0 || g.Lq == 0) return CUSTMA_OK;
    if ((rc = check_grid(g)) || (rc = check_space(geo, g, CUSTMA_MATCH_ATTENTION, workspace, workspace_bytes))) return rc;
    if (!q || !out || (g.Lk > 0 && (!k || !v))) return refuse(CUSTMA_E_NULL, "null pointer argument");
    if (unaligned(q) || unaligned(k) || unaligned(v) || unaligned(out) || unaligned(low))
        return refuse(CUSTMA_E_ARG, "rows must be 16-byte aligned");
    Carve c{(char*)workspace};
    FwdSpace w;
    carve_fwd(g, false, c, &w);
    FwdOut o{};
    o.out = out;
    o.low = geo->out_f32 ? nullptr : low;
    o.lse = lse;
    o.part = w.part;
    o.part_ml = w.part_ml;
    return ran(run_fwd(g, geo->dtype, geo->out_f32 != 0, q, k, v, o, (hipStream_t)stream), "match_attention");
}

int custma_match_attention_backward(const custma_match_geo* geo, const void* q, const void* k, const void* v,
                                    const void* out, const void* low, const float* lse, const void* grad_out,
                                    void* grad_q, void* grad_k, void* grad_v, float* unit, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    MatchGeo g;
    int rc = make_match(geo, CUSTMA_MATCH_ATTENTION_BACKWARD, &g);
    if (rc) return rc;
    if (g.B == 0 || (!grad_q && !grad_k && !grad_v)) return CUSTMA_OK;
    if ((rc = check_grid(g)) || (rc = check_space(geo, g, CUSTMA_MATCH_ATTENTION_BACKWARD, workspace, workspace_bytes))) return rc;
    if ((g.Lq > 0 && (!q || !out || !lse || !grad_out || (!low && !geo->out_f32))) || (g.Lk > 0 && (!k || !v)))
        return refuse(CUSTMA_E_NULL, "null pointer argument");
    if (unaligned(q) || unaligned(k) || unaligned(v) || unaligned(out) || unaligned(low) || unaligned(grad_out) ||
        unaligned(grad_q) || unaligned(grad_k) || unaligned(grad_v))
        return refuse(CUSTMA_E_ARG, "rows must be 16-byte aligned");
    if (unit && !geo->out_f32) return refuse(CUSTMA_E_ARG, "unit needs a float32 output");
    hipStream_t s = (hipStream_t)stream;
    Carve c{(char*)workspace};
    BwdSpace w;
    carve_bwd(g, geo->out_f32 != 0, c, &w);
    const Dims d = dims(g);
    BwdArgs a{};
    a.q = q, a.k = k, a.v = v;
    a.gq = grad_q, a.gk = grad_k, a.gv = grad_v;
    a.go = grad_out;
    if (g.Lq > 0) {
        if (geo->out_f32) {
            float* scale = unit ? unit : w.scale;
            if ((rc = ran(launch_match_narrow((const float*)grad_out, d.rows * g.Cv, geo->dtype, w.go16, scale, w.partials, s), "match_attention_backward"))) return rc;
            a.go = w.go16;
            a.factor = unit ? nullptr : scale;
        }
    }
    return ran(run_bwd(g, geo->dtype, a, w, lse, out, geo->out_f32 != 0, low, s), "match_attention_backward");
}

int custma_match_entropy(const custma_match_geo* geo, const void* q, const void* k, const int64_t* target, float* loss,
                         float* lse, float* total, void* workspace, size_t workspace_bytes, void* stream) {
    MatchGeo g;
    int rc = make_match(geo, CUSTMA_MATCH_ENTROPY, &g);
    if (rc) return rc;
    hipStream_t s = (hipStream_t)stream;
    const int64_t rows = (int64_t)g.B * g.Lq;
    if (rows == 0 && !total) return CUSTMA_OK;
    if ((rc = check_grid(g)) || (rc = check_space(geo, g, CUSTMA_MATCH_ENTROPY, workspace, workspace_bytes))) return rc;
    if (rows > 0 && (!q || !target || !loss || !lse || (g.Lk > 0 && !k))) return refuse(CUSTMA_E_NULL, "null pointer argument");
    if (unaligned(q) || unaligned(k)) return refuse(CUSTMA_E_ARG, "rows must be 16-byte aligned");
    Carve c{(char*)workspace};
    FwdSpace w{};
    if (rows > 0) {
        carve_fwd(g, true, c, &w);
        FwdOut o{};
        o.lse = lse;
        o.loss = loss;
        o.target = target;
        o.part_ml = w.part_ml;
        const hipError_t e = g.C > kMatchMaxC ? launch_wide_fwd(g, geo->dtype, q, k, o, s)
                                              : run_fwd(g, geo->dtype, false, q, k, nullptr, o, s);
        if ((rc = ran(e, "match_entropy"))) return rc;
    } else {
        w.partials = (double*)workspace;
    }
    if (total) return ran(launch_match_total(loss, target, g, rows, total, w.partials, s), "match_entropy");
    return CUSTMA_OK;
}

int custma_match_entropy_backward(const custma_match_geo* geo, const void* q, const void* k, const int64_t* target,
                                  const float* lse, const float* weight, const float* factor, void* grad_q,
                                  void* grad_k, float* unit, void* workspace, size_t workspace_bytes, void* stream) {
    MatchGeo g;
    int rc = make_match(geo, CUSTMA_MATCH_ENTROPY_BACKWARD, &g);
    if (rc) return rc;
    const bool wide = g.C > kMatchMaxC;
    if (g.B == 0 || (!grad_q && !grad_k)) return CUSTMA_OK;
    if (wide && (g.Lq == 0 || g.Lk == 0)) return refuse(CUSTMA_E_ARG, "empty queries or classes have no gradient kernel for wide vectors");
    if ((rc = check_grid(g)) || (rc = check_space(geo, g, CUSTMA_MATCH_ENTROPY_BACKWARD, workspace, workspace_bytes))) return rc;
    if ((g.Lq > 0 && (!q || !target || !lse)) || (g.Lk > 0 && !k)) return refuse(CUSTMA_E_NULL, "null pointer argument");
    if (unaligned(q) || unaligned(k) || unaligned(grad_q) || unaligned(grad_k)) return refuse(CUSTMA_E_ARG, "rows must be 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    BwdArgs a{};
    a.q = q, a.k = k, a.lse = lse, a.target = target, a.factor = factor;
    a.gq = grad_q, a.gk = grad_k;
    Carve c{(char*)workspace};
    const WeightSpace ws = carve_weights(g, c);
    if (weight || unit) {
        float* scale = unit ? unit : ws.scale;
        if ((rc = ran(launch_match_weights(weight, dims(g).rows, factor, ws.weight, scale, ws.partials, s), "match_entropy_backward"))) return rc;
        if (weight) a.weight = ws.weight;
        a.factor = unit ? nullptr : scale;
    }
    if (wide) return ran(launch_wide_bwd(g, geo->dtype, a, c.base + c.at, s), "match_entropy_backward");
    BwdSpace w;
    carve_bwd(g, false, c, &w);
    return ran(run_bwd(g, geo->dtype, a, w, lse, nullptr, false, nullptr, s), "match_entropy_backward");
}

static int check_desc(int32_t image_dtype, int64_t H, int64_t W, int32_t k, int32_t out_dtype) {
    if (image_dtype != CUSTMA_F32 && image_dtype != CUSTMA_F16)
        return refuse(CUSTMA_E_ARG, "unsupported image dtype code %d (float32=0, float16=1)", image_dtype);
    if (out_dtype != CUSTMA_F16 && out_dtype != CUSTMA_BF16)
        return refuse(CUSTMA_E_ARG, "unsupported descriptor dtype code %d (float16=1, bfloat16=2)", out_dtype);
    if (H < 0 || W < 0) return refuse(CUSTMA_E_ARG, "negative image size");
    if (k < 1 || k > desc_max_kernel())
        return refuse(CUSTMA_E_ARG, "descriptors need kernel_size in [1, %d], got %d", desc_max_kernel(), k);
    const int64_t top = (int64_t)1 << 31;  // clamped, the product stays within 64 bits
    return check_blocks(cdiv(at_most(H, top), 4) * cdiv(at_most(W, top), 64));
}

int custma_descriptors(const void* image, int32_t image_dtype, int64_t H, int64_t W, int32_t kernel_size,
                       int32_t out_dtype, void* out, float* stats, void* stream) {
    const int rc = check_desc(image_dtype, H, W, kernel_size, out_dtype);
    if (rc) return rc;
    if (H == 0 || W == 0) return CUSTMA_OK;
    if (!image || !out) return refuse(CUSTMA_E_NULL, "null pointer argument");
    if (unaligned(out)) return refuse(CUSTMA_E_ARG, "rows must be 16-byte aligned");
    return ran(launch_desc(image, image_dtype, H, W, kernel_size, out_dtype, out, stats, (hipStream_t)stream),
               "descriptors");
}

int custma_descriptors_backward(const void* image, int32_t image_dtype, int64_t H, int64_t W, int32_t kernel_size,
                                int32_t out_dtype, const float* stats, const void* grad, const float* factor, void* image_grad,
                                void* stream) {
    const int rc = check_desc(image_dtype, H, W, kernel_size, out_dtype);
    if (rc) return rc;
    if (H == 0 || W == 0) return CUSTMA_OK;
    if (!image || !stats || !grad || !image_grad) return refuse(CUSTMA_E_NULL, "null pointer argument");
    if (unaligned(grad)) return refuse(CUSTMA_E_ARG, "rows must be 16-byte aligned");
    return ran(launch_desc_bwd(image, image_dtype, H, W, kernel_size, out_dtype, stats, grad, factor, image_grad,
                               (hipStream_t)stream),
               "descriptors_backward");
}

}  // extern "C"

// dorado_amd/csrc/ops_attention.hip — host half of mibc_attention: checks, choice of the kernel and of the split over the keys.
#include "ops_attention.h"

#include <math.h>

static int att_check(const mibc_attention_args &a) {
    if (a.type != MIBC_TYPE_F16 && a.type != MIBC_TYPE_BF16) return op_refuse(MIBC_NOT_SUPPORTED, "attention: type must be f16 or bf16");
    if (a.head_dim != 32 && a.head_dim != 64 && a.head_dim != 96 && a.head_dim != 128)
        return op_refuse(MIBC_NOT_SUPPORTED, "attention: head_dim must be 32, 64, 96 or 128");
    if (a.batch < 0 || a.q_tokens < 0 || a.k_tokens < 0 || a.heads < 1 || a.kv_heads < 1)
        return op_refuse(MIBC_ERR_ARG, "attention: negative size, or no heads");
    if (a.heads % a.kv_heads != 0) return op_refuse(MIBC_ERR_ARG, "attention: heads must be a multiple of kv_heads");
    if (!(a.scale > 0.0f) || !(a.scale <= 1e30f)) return op_refuse(MIBC_ERR_ARG, "attention: scale must be positive and finite");
    if (!(a.softcap >= 0.0f) || !(a.softcap <= 1e30f)) return op_refuse(MIBC_ERR_ARG, "attention: softcap must be 0 (none) or positive and finite");
    if (a.softcap > 0.0f && !(3.0f * a.scale / a.softcap <= 3e38f)) return op_refuse(MIBC_ERR_ARG, "attention: softcap too small for this scale");
    if (a.softcap > 0.0f && !(a.softcap / a.scale <= 3e37f)) return op_refuse(MIBC_ERR_ARG, "attention: softcap too large for this scale");
    // a slope is held in the scores' unit: slope / scale, or slope / (2 softcap)
    if (a.slopes != nullptr && (a.scale < 1e-18f || (a.softcap > 0.0f && a.softcap < 1e-18f)))
        return op_refuse(MIBC_ERR_ARG, "attention: slopes need a scale and a softcap of at least 1e-18");
    if (a.reserved != 0) return op_refuse(MIBC_ERR_ARG, "attention: reserved must be 0");
    const int64_t big = (int64_t)1 << 28;     // positions, and distances between them, stay far inside 32 bits
    if (a.q_tokens > big || a.k_tokens > big || (int64_t)a.q_tokens * (a.heads / a.kv_heads) > big ||
        (int64_t)a.batch * a.kv_heads > big || (a.q_start != MIBC_ATTN_END && (a.q_start > big || a.q_start < -big)))
        return op_refuse(MIBC_NOT_SUPPORTED, "attention: more than 2^28 tokens, rows or heads");
    if (a.doc_offsets != nullptr) {
        if (a.batch != 1 || a.q_tokens != a.k_tokens || a.k_len != nullptr || a.q_start != MIBC_ATTN_END)
            return op_refuse(MIBC_ERR_ARG, "attention: documents need batch 1, q_tokens == k_tokens, no k_len and no q_start");
        if (a.n_docs < 0 || a.n_docs > big) return op_refuse(MIBC_ERR_ARG, "attention: n_docs");
    } else if (a.n_docs != 0) {
        return op_refuse(MIBC_ERR_ARG, "attention: n_docs without doc_offsets");
    }
    if (a.batch == 0 || a.q_tokens == 0) return MIBC_OK;
    if (a.q == nullptr || a.out == nullptr || (a.k_tokens > 0 && (a.k == nullptr || a.v == nullptr)))
        return op_refuse(MIBC_ERR_ARG, "attention: null pointer");
    const int64_t qs[3] = {a.batch, a.q_tokens, a.heads}, ks[3] = {a.batch, a.k_tokens, a.kv_heads};
    for (int d = 0; d < 3; ++d) {
        if (a.q_stride[d] < 0 || a.k_stride[d] < 0 || a.v_stride[d] < 0) return op_refuse(MIBC_ERR_ARG, "attention: negative stride");
        if (qs[d] > 1 && a.out_stride[d] < a.head_dim) return op_refuse(MIBC_ERR_ARG, "attention: output heads overlap");
        if ((qs[d] > 1 && (a.q_stride[d] % 8 != 0 || a.out_stride[d] % 8 != 0)) || (ks[d] > 1 && (a.k_stride[d] % 8 != 0 || a.v_stride[d] % 8 != 0)))
            return op_refuse(MIBC_NOT_SUPPORTED, "attention: strides must be multiples of 8 elements");
    }
    // a tile's rows are reached through 32-bit offsets from its first one
    if (a.k_tokens > 1 && (a.k_stride[1] > (1 << 24) || a.v_stride[1] > (1 << 24)))
        return op_refuse(MIBC_NOT_SUPPORTED, "attention: key and value tokens at most 2^24 elements apart");
    if (!op_aligned(a.q, 16) || !op_aligned(a.out, 16) || !op_aligned(a.k, 16) || !op_aligned(a.v, 16))
        return op_refuse(MIBC_NOT_SUPPORTED, "attention: pointers must be aligned to 16 bytes");
    if (!op_aligned(a.lse, 4) || !op_aligned(a.k_len, 4) || !op_aligned(a.prefix, 4) || !op_aligned(a.doc_offsets, 4) || !op_aligned(a.slopes, 4))
        return op_refuse(MIBC_ERR_ARG, "attention: pointer not aligned to its type");
    return MIBC_OK;
}

struct AttPlan {
    bool tokens;     // at most 16 rows per (batch, key head) pair
    int tiles, splits;
};
static AttPlan att_plan(const mibc_attention_args &a) {
    const int64_t rows = (int64_t)a.q_tokens * (a.heads / a.kv_heads), pairs = (int64_t)a.batch * a.kv_heads;
    AttPlan p;
    p.tokens = rows <= 16;
    const int tile = p.tokens ? 16 : 128;
    p.tiles = (int)((rows + tile - 1) / tile);
    // keys a row can see at most
    int64_t keys = a.k_tokens;
    if (a.window_back >= 0 && a.window_ahead >= 0 && a.prefix == nullptr) {
        const int64_t w = (int64_t)a.window_back + a.window_ahead + 1 + tile;
        keys = keys < w ? keys : w;
    }
    const int64_t groups = p.tiles * pairs;
    int64_t splits = 1;
    if (p.tokens) {
        // the smallest number of parts that fills whole rounds of one workgroup per CU to nine tenths (one token over 131072 keys,
        // 2 key heads: 128 parts 34 us, 255 parts 41, 64 parts 38; 32 pairs x 4096 keys: 8 parts 17 us, 4 parts 20, 32 parts 20);
        // rows of different lengths: five or more parts per pair even out the lengths (48 x 8 pairs of 2048 .. 8192 keys: 191 us
        // against 248 unsplit).  At least four steps of 32 keys for each of the four waves: a
        // shorter part costs more in the second launch than it saves (512 keys: 9.0 us whole, 13.9 in two)
        const int64_t most = keys / 512 < 255 ? keys / 512 : 255, cus = 256;
        double best = 0.0;
        for (int64_t s = 1; s <= most; ++s) {
            const int64_t all = groups * s;
            const double full = (double)all / (double)((all + cus - 1) / cus * cus);
            if (full > best + 1e-9) {
                best = full;
                splits = s;
            }
            if (best >= 0.9) break;
        }
        if (a.k_len != nullptr && splits * groups < 2048) splits = 2048 / groups < most ? 2048 / groups : most;
    } else {
        // tiles: a workgroup per CU (64 rows of 4 heads each over 16384 keys, 8 tiles: 32 parts 26 us, 64 parts 30, 16 parts 32), two
        // where a tile is half empty and reading the keys is what takes the time (8 x 8 pairs of 32 rows over 8192 keys: 8 parts
        // 58 us, 4 parts 69), and at least four tiles of 64 keys in a part
        const int64_t want = rows <= 64 ? 512 : 256;
        if (groups < want) splits = want / groups;
        if (splits > keys / 256) splits = keys / 256;
    }
    if (splits > 255) splits = 255;
    p.splits = splits < 1 ? 1 : (int)splits;
    return p;
}

static uint64_t att_room(const mibc_attention_args &a, const AttPlan &p) {
    return p.splits == 1 ? 0 : (uint64_t)a.batch * a.heads * a.q_tokens * p.splits * (a.head_dim + 1) * 4;
}
static int att_check_plan(const mibc_attention_args &a, const AttPlan &p) {
    if ((int64_t)a.batch * a.kv_heads * p.tiles * p.splits > 0x7fffffff) return op_refuse(MIBC_NOT_SUPPORTED, "attention: too many row tiles");
    const uint64_t need = att_room(a, p);
    if (need != 0 && (a.workspace == nullptr || a.workspace_bytes < need))
        return op_refuse(MIBC_ERR_ARG, "attention: workspace smaller than mibc_attention_workspace says");
    if (need != 0 && !op_aligned(a.workspace, 16)) return op_refuse(MIBC_ERR_ARG, "attention: workspace must be aligned to 16 bytes");
    // a workgroup writes its rows while others still read
    auto span = [&](const void *x, int64_t tokens, int64_t heads, const int64_t *s) {
        return op_span(x, a.head_dim * 2, a.batch, s[0] * 2, tokens, s[1] * 2, heads, s[2] * 2);
    };
    const OpSpan q = span(a.q, a.q_tokens, a.heads, a.q_stride), k = span(a.k, a.k_tokens, a.kv_heads, a.k_stride),
                 v = span(a.v, a.k_tokens, a.kv_heads, a.v_stride), out = span(a.out, a.q_tokens, a.heads, a.out_stride);
    if (!op_plain(out)) return op_refuse(MIBC_ERR_ARG, "attention: output heads overlap");
    if (!op_apart(out, k) || !op_apart(out, v) || (!op_same(out, q) && !op_apart(out, q)))
        return op_refuse(MIBC_ERR_ARG, "attention: out may be q, but not k or v, nor overlap any of them otherwise");
    const OpSpan lse = op_span(a.lse, (int64_t)a.batch * a.heads * a.q_tokens * 4), room = op_span(need ? a.workspace : nullptr, (int64_t)need);
    const OpSpan small[4] = {op_span(a.k_len, (int64_t)a.batch * 4), op_span(a.prefix, (int64_t)(a.doc_offsets ? a.n_docs : a.batch) * 4),
                             op_span(a.doc_offsets, ((int64_t)a.n_docs + 1) * 4), op_span(a.slopes, (int64_t)a.heads * 4)};
    bool fine = op_apart(out, lse) && op_apart(out, room) && op_apart(lse, room);
    for (const OpSpan *x : {&q, &k, &v, &small[0], &small[1], &small[2], &small[3]}) fine = fine && op_apart(lse, *x) && op_apart(room, *x);
    for (const OpSpan &x : small) fine = fine && op_apart(out, x);
    if (!fine) return op_refuse(MIBC_ERR_ARG, "attention: out, lse and workspace may not overlap another operand");
    return MIBC_OK;
}

extern "C" uint64_t mibc_attention_workspace(const mibc_attention_args *a) {
    if (a == nullptr || att_check(*a) != MIBC_OK || a->batch == 0 || a->q_tokens == 0) return 0;
    return att_room(*a, att_plan(*a));
}

static int att_run(hipStream_t s, const mibc_attention_args &a, const AttPlan &plan) {
    AttArgs p{};
    p.a = a;
    p.group = a.heads / a.kv_heads;
    p.rows = a.q_tokens * p.group;
    p.pairs = a.batch * a.kv_heads;
    p.tiles = plan.tiles;
    p.splits = plan.splits;
    p.by_pairs.set((unsigned)p.pairs);
    p.by_splits.set((unsigned)p.splits);
    p.by_tiles.set((unsigned)p.tiles);
    p.by_kv.set((unsigned)a.kv_heads);
    p.by_group.set((unsigned)p.group);
    p.back = a.window_back >= 0 && a.window_back < 1 << 30 ? a.window_back : -1;
    p.ahead = a.window_ahead >= 0 && a.window_ahead < 1 << 30 ? a.window_ahead : -1;
    p.scale2 = a.scale * 1.4426950408889634f;
    // tiles: caps up to 64 take the form of fewer instructions, whose error grows with the cap (causal 16384 x 16 heads of 128: 1210 us,
    // the other form 1788, no cap 1046).  Single tokens are bound by bytes: 285 us either way and without a cap (48 x 8 pairs x 8192)
    if (a.softcap > 64.0f || (a.softcap > 0.0f && plan.tokens)) {
        p.cap = ATT_FAR;
        p.cap_in = a.scale / a.softcap;
        p.cap_out = a.softcap / a.scale;
    } else if (a.softcap > 0.0f) {
        p.cap = ATT_NEAR;
        p.cap_in = 2.0f * a.scale / a.softcap * 1.4426950408889634f;
        p.cap_out = a.softcap * 1.4426950408889634f;
    }
    if (plan.splits > 1) {
        p.part_o = (float *)a.workspace;
        p.part_l = p.part_o + (uint64_t)p.pairs * p.rows * p.splits * a.head_dim;
    }
    p.groups = (unsigned)((int64_t)p.pairs * p.tiles * p.splits);
    p.order = (a.window_ahead != 0 && p.pairs % 8 == 0) ? 1 : 0;
    // heads of 64 or 192 bytes share 128-byte lines with their neighbours, which two XCDs would both fetch (32 x 4 pairs over 8192 keys
    // of 32: 45 -> 28 us, 64 x 1024 windows of 256 keys, 8 heads of 32: 72 -> 53, of 96: 149 -> 132; nothing at 64 and 128)
    p.twin = a.head_dim % 64 != 0 && a.kv_heads % 2 == 0 && p.pairs % 16 == 0 && a.k_stride[2] == a.head_dim;
    switch (a.head_dim) {
        case 32: return mibc_att_launch_32(s, p, plan.tokens);
        case 64: return mibc_att_launch_64(s, p, plan.tokens);
        case 96: return mibc_att_launch_96(s, p, plan.tokens);
        default: return mibc_att_launch_128(s, p, plan.tokens);
    }
}

// launch on a stream of the current device (the engine's own path); checks included.  whole: the keys are not split, so there is
// no workspace (the engine's batches fill the device)
int mibc_launch_attention(hipStream_t s, const mibc_attention_args &a, bool whole) {
    if (const int rc = att_check(a)) return rc;
    if (a.batch == 0 || a.q_tokens == 0) return MIBC_OK;
    AttPlan plan = att_plan(a);
    if (whole) plan.splits = 1;
    if (const int rc = att_check_plan(a, plan)) return rc;
    return att_run(s, a, plan);
}

extern "C" int mibc_attention(int device, void *stream, const mibc_attention_args *a) {
    if (a == nullptr) return op_refuse(MIBC_ERR_ARG, "attention: null arguments");
    if (const int rc = att_check(*a)) return rc;
    if (a->batch == 0 || a->q_tokens == 0) return MIBC_OK;
    const AttPlan plan = att_plan(*a);
    if (const int rc = att_check_plan(*a, plan)) return rc;
    OpDevice d(device);
    if (d.rc != hipSuccess) return op_hip(d.rc, "attention: device");
    return att_run((hipStream_t)stream, *a, plan);
}

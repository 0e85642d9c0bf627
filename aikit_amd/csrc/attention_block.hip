// attention_block.hip -- entry points of what stands in an encoder's attention block beside the linears of
// enchip.hip: head norms with rotation, attention with a relative position bias, low-rank adapters.
#include "context.h"

#include "adapters.h"
#include "attention_bias.h"
#include "gemm_pieces.h"
#include "head_norm.h"

using namespace enchip_host;

extern "C" {

// ---------------------------------------------------------------------------- head norms

int enchip_head_norm_rope_rows_dev(enchip_ctx *ctx, enchip_rope h, int layout, const float *d_x, int64_t ldx, float *d_y,
                                   int64_t ldy, int64_t nseq, int64_t L, int64_t q_heads, int64_t k_heads, int64_t head_dim,
                                   const float *d_q_gain, const float *d_k_gain, double eps, const int32_t *d_pos, int64_t pos0,
                                   void *stream) {
    if (!ctx) return ENCHIP_ERR_ARG;
    std::lock_guard<std::mutex> g(ctx->mu);
    Rope r;
    if (h != 0) {
        auto it = ctx->ropes.find(h);
        if (it == ctx->ropes.end()) return fail(ctx, ENCHIP_ERR_HANDLE, "unknown rope handle %llu", (unsigned long long)h);
        r = it->second;
        if (layout != ENCHIP_ROPE_HALF && layout != ENCHIP_ROPE_INTERLEAVED)
            return fail(ctx, ENCHIP_ERR_ARG, "head_norm: bad layout %d", layout);
        if (!d_pos && (pos0 < -((int64_t)1 << 31) || pos0 > ((int64_t)1 << 31)))
            return fail(ctx, ENCHIP_ERR_ARG, "head_norm: pos0=%lld past 32 bits", (long long)pos0);
    } else {
        d_pos = nullptr;
        pos0 = 0;
        layout = ENCHIP_ROPE_HALF;
    }
    const int64_t max_hd = 2 * enchip::ROPE_MAX_PAIRS;
    if (nseq < 0 || L < 0 || q_heads < 0 || k_heads < 0 || q_heads > 65536 || k_heads > 65536 - q_heads || head_dim < 1 ||
        head_dim < 2 * r.n || head_dim > max_hd || (q_heads + k_heads) * head_dim > ((int64_t)1 << 20) || nseq > INT32_MAX ||
        L > INT32_MAX || nseq * L > INT32_MAX || ldx < (q_heads + k_heads) * head_dim || ldy < (q_heads + k_heads) * head_dim)
        return fail(ctx, ENCHIP_ERR_ARG,
                    "head_norm: bad shape nseq=%lld L=%lld q_heads=%lld k_heads=%lld head_dim=%lld (%lld rotated, at most %lld) "
                    "ldx=%lld ldy=%lld",
                    (long long)nseq, (long long)L, (long long)q_heads, (long long)k_heads, (long long)head_dim,
                    (long long)(2 * r.n), (long long)max_hd, (long long)ldx, (long long)ldy);
    if (!(eps >= 0x1p-100 && eps <= 0x1p100)) return fail(ctx, ENCHIP_ERR_ARG, "head_norm: eps %g is not from 2^-100 to 2^100", eps);
    if (d_x == d_y && ldx != ldy)
        return fail(ctx, ENCHIP_ERR_ARG, "head_norm: in place needs one pitch, not %lld and %lld", (long long)ldx, (long long)ldy);
    const int64_t heads = q_heads + k_heads, rows = nseq * L;
    if (rows == 0 || heads == 0) return ENCHIP_OK;
    if (!d_x || !d_y || (q_heads > 0 && !d_q_gain) || (k_heads > 0 && !d_k_gain))
        return fail(ctx, ENCHIP_ERR_ARG, "head_norm: null pointer");
    HIP_TRY(ctx, hipSetDevice(ctx->device));
    hipStream_t s = stream ? (hipStream_t)stream : ctx->stream;
    const bool inter = layout == ENCHIP_ROPE_INTERLEAVED;
    const int64_t rot = 2 * r.n;
    // elements that an access holds: whole parts of a slot, aligned (rope.h's 16 bytes against 4: a third of the time)
    auto fits = [&](int64_t n) {
        return (inter ? rot % (2 * n) == 0 : r.n % n == 0) && head_dim % n == 0 && ldx % n == 0 && ldy % n == 0 &&
               (uintptr_t)d_x % (4 * n) == 0 && (uintptr_t)d_y % (4 * n) == 0;
    };
    const int v = fits(4) ? 4 : fits(2) ? 2 : 1;
    enchip::HeadNorm p;
    p.gain_q = d_q_gain ? d_q_gain : d_k_gain;
    p.gain_k = d_k_gain ? d_k_gain : d_q_gain;
    p.eps = eps;
    p.inv_hd = 1.0 / (double)head_dim;
    p.q_heads = (int)q_heads;
    p.hd = (int)head_dim;
    p.r = (int)rot;
    p.turned = (int)(r.n / v);
    p.slots = p.turned + (int)((head_dim - rot + 2 * v - 1) / (2 * v));
    p.lanes = 1;
    while (p.lanes < 64 && p.lanes < p.slots) p.lanes *= 2;
    const int need = (p.slots + p.lanes - 1) / p.lanes, it = need <= 1 ? 1 : need <= 2 ? 2 : need <= 4 ? 4 : 8;
    // rows of a workgroup: one pass of its lanes, two where the positions come from memory and the angles wait for
    // them (64 x 512 rows of 24 heads of 64 75 us against 80 with two passes and 82 with three; 20011 rows of 20 heads
    // of 128 with positions 93.5, 89 and 93), while a few workgroups a CU are left
    const int64_t passes = d_pos ? 2 : 1, pass = 256 / p.lanes * (it >= 4 ? 1 : 4 / it);
    const int64_t by_items = std::max<int64_t>(1, passes * pass / heads), by_rows = std::max<int64_t>(1, rows / (4 * ctx->num_cus));
    const int64_t by_angles = r.n ? (int64_t)enchip::ROPE_CS / r.n : 64;
    const int tr = (int)std::min({by_items, by_rows, by_angles, (int64_t)64});
    for (int64_t r0 = 0; r0 < rows; r0 += kRowChunk) {
        const int64_t n = std::min(kRowChunk, rows - r0);
#define HN_CALL(I, V, IT)                                                                                                   \
    hipLaunchKernelGGL((enchip::head_norm_rope<I, V, IT>), dim3((unsigned)((n + tr - 1) / tr)), dim3(256), 0, s, d_x + r0 * ldx, \
                       ldx, d_y + r0 * ldy, ldy, p, r.d_turns, r.mscale, d_pos ? d_pos + r0 : nullptr, pos0, r0, (int)L, n, tr, \
                       fast_div(heads))
#define HN_V(I)                                     \
    do {                                            \
        if (v == 4 && it == 1) HN_CALL(I, 4, 1);    \
        else if (v == 4) HN_CALL(I, 4, 2);          \
        else if (v == 2 && it == 1) HN_CALL(I, 2, 1); \
        else if (v == 2 && it == 2) HN_CALL(I, 2, 2); \
        else if (v == 2) HN_CALL(I, 2, 4);          \
        else if (it == 1) HN_CALL(I, 1, 1);         \
        else if (it == 2) HN_CALL(I, 1, 2);         \
        else if (it == 4) HN_CALL(I, 1, 4);         \
        else HN_CALL(I, 1, 8);                      \
    } while (0)
        if (inter) HN_V(true);
        else HN_V(false);
#undef HN_V
#undef HN_CALL
    }
    return check_launch(ctx, "head_norm_rope");
}

// ---------------------------------------------------------------------------- relative position bias

}  // extern "C"

namespace {

constexpr int64_t kMaxReach = (int64_t)1 << 20;

// Expands table[buckets][heads] over the distances -reach .. reach (bucket(d) within [0, buckets)) into a handle.
template <typename F>
int add_relpos(enchip_ctx *ctx, const float *table, int64_t buckets, int64_t heads, int64_t reach, F bucket, enchip_relpos *out) {
    for (int64_t i = 0; i < buckets * heads; ++i)
        if (!(table[i] <= 0x1p100f) || (table[i] < -0x1p100f && !std::isinf(table[i])))
            return fail(ctx, ENCHIP_ERR_ARG, "relpos: value %g of bucket %lld, head %lld is neither -infinity nor within 2^100 of 0",
                        (double)table[i], (long long)(i / heads), (long long)(i % heads));
    const int64_t width = 2 * reach + 1;
    std::vector<float> all;
    try {
        all.resize((size_t)(heads * width));
    } catch (const std::exception &) {
        return fail(ctx, ENCHIP_ERR_OOM, "relpos: out of host memory");
    }
    for (int64_t d = -reach; d <= reach; ++d) {
        const float *row = table + bucket(d) * heads;
        for (int64_t i = 0; i < heads; ++i) all[(size_t)(i * width + d + reach)] = (float)((double)row[i] * 1.4426950408889634074);
    }
    HIP_TRY(ctx, hipSetDevice(ctx->device));
    RelPos r;
    r.heads = heads;
    r.reach = reach;
    size_t cap = 0;
    if (int rc = ensure(ctx, &r.d_table, &cap, all.size() * sizeof(float), false)) return rc;
    const hipError_t e = hipMemcpy(r.d_table, all.data(), all.size() * sizeof(float), hipMemcpyHostToDevice);
    if (e != hipSuccess) {
        (void)hipFree(r.d_table);
        return fail(ctx, ENCHIP_ERR_HIP, "relpos upload: %s", hipGetErrorString(e));
    }
    try {
        ctx->relpos[ctx->next_handle] = r;
    } catch (const std::bad_alloc &) {
        (void)hipFree(r.d_table);
        return fail(ctx, ENCHIP_ERR_OOM, "relpos: out of host memory");
    }
    *out = ctx->next_handle++;
    return ENCHIP_OK;
}

int check_relpos(enchip_ctx *ctx, const float *table, int64_t buckets, int64_t heads, int64_t reach, enchip_relpos *out) {
    if (!out) return fail(ctx, ENCHIP_ERR_ARG, "relpos: out is NULL");
    *out = 0;
    if (buckets < 1 || buckets > ((int64_t)1 << 22) || heads < 1 || heads > 65535 || reach < 0 || reach > kMaxReach ||
        heads * (2 * reach + 1) > ((int64_t)1 << 28))
        return fail(ctx, ENCHIP_ERR_ARG, "relpos: bad shape buckets=%lld heads=%lld reach=%lld", (long long)buckets,
                    (long long)heads, (long long)reach);
    if (!table) return fail(ctx, ENCHIP_ERR_ARG, "relpos: null pointer");
    return ENCHIP_OK;
}

}  // namespace

extern "C" {

int enchip_relpos_create(enchip_ctx *ctx, const float *table, int64_t buckets, int64_t heads, int64_t max_distance,
                         enchip_relpos *out) {
    if (!ctx) return ENCHIP_ERR_ARG;
    std::lock_guard<std::mutex> g(ctx->mu);
    if (int rc = check_relpos(ctx, table, buckets, heads, max_distance, out)) return rc;
    const int64_t half = buckets / 2, exact = half / 2;
    if (buckets % 2 != 0 || buckets < 4 || max_distance <= exact)
        return fail(ctx, ENCHIP_ERR_ARG, "relpos: %lld buckets (even, at least 4) up to distance %lld (past %lld)",
                    (long long)buckets, (long long)max_distance, (long long)exact);
    const double per = (double)(half - exact) / std::log((double)max_distance / (double)exact);
    return add_relpos(ctx, table, buckets, heads, max_distance, [&](int64_t d) {
        const int64_t n = d < 0 ? -d : d;
        int64_t b = n;
        if (n >= exact)
            b = std::min<int64_t>(half - 1, exact + (int64_t)std::floor(std::log((double)n / (double)exact) * per + 1e-9));
        return d > 0 ? half + b : b;
    }, out);
}

int enchip_relpos_create_map(enchip_ctx *ctx, const float *table, int64_t buckets, int64_t heads, const int32_t *bucket_of,
                             int64_t reach, enchip_relpos *out) {
    if (!ctx) return ENCHIP_ERR_ARG;
    std::lock_guard<std::mutex> g(ctx->mu);
    if (int rc = check_relpos(ctx, table, buckets, heads, reach, out)) return rc;
    if (!bucket_of) return fail(ctx, ENCHIP_ERR_ARG, "relpos: null pointer");
    for (int64_t i = 0; i <= 2 * reach; ++i)
        if (bucket_of[i] < 0 || bucket_of[i] >= buckets)
            return fail(ctx, ENCHIP_ERR_ARG, "relpos: distance %lld has bucket %d of %lld", (long long)(i - reach), bucket_of[i],
                        (long long)buckets);
    return add_relpos(ctx, table, buckets, heads, reach, [&](int64_t d) { return (int64_t)bucket_of[d + reach]; }, out);
}

int enchip_relpos_release(enchip_ctx *ctx, enchip_relpos h) {
    if (!ctx) return ENCHIP_ERR_ARG;
    std::lock_guard<std::mutex> g(ctx->mu);
    auto it = ctx->relpos.find(h);
    if (it == ctx->relpos.end()) return fail(ctx, ENCHIP_ERR_HANDLE, "unknown relpos handle %llu", (unsigned long long)h);
    HIP_TRY(ctx, hipSetDevice(ctx->device));
    HIP_TRY(ctx, hipStreamSynchronize(ctx->stream));
    (void)hipFree(it->second.d_table);
    ctx->relpos.erase(it);
    return ENCHIP_OK;
}

}  // extern "C"

namespace {

// Launches fn over (query blocks of 2^qs rows) x (head sets), in chunks of sequences, or with spans of query blocks, whose
// threads are numbered in 32 bits. p.order, and parts, are one launch (attention_plan).
int launch_attention_bias(enchip_ctx *ctx, void (*fn)(enchip::AttnBias), int lds, int threads, int qs, enchip::AttnBias p, hipStream_t s) {
    const std::pair<const void *, size_t> key(reinterpret_cast<const void *>(fn), (size_t)lds);
    if (std::find(ctx->lds_set.begin(), ctx->lds_set.end(), key) == ctx->lds_set.end()) {
        HIP_TRY(ctx, hipFuncSetAttribute(key.first, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
        ctx->lds_set.push_back(key);
    }
    const int64_t qr = (int64_t)1 << qs, sets = (int64_t)(p.heads >> p.share) * p.parts;
    const int64_t per = p.spans ? p.L / qr + p.nseq : (p.L + qr - 1) / qr;
    const int64_t most = (((int64_t)1 << 32) - 1) / threads / sets;
    if (p.order) {
        hipLaunchKernelGGL(fn, dim3((unsigned)round_up(per * sets, 32)), dim3((unsigned)threads), (size_t)lds, s, p);
        return check_launch(ctx, "attention_bias");
    }
    if (p.spans) {
        for (int64_t b0 = 0; b0 < per; b0 += most) {
            p.block0 = (int)b0;
            hipLaunchKernelGGL(fn, dim3((unsigned)(std::min(most, per - b0) * sets)), dim3((unsigned)threads), (size_t)lds, s, p);
        }
        return check_launch(ctx, "attention_bias");
    }
    if (per > most)
        return fail(ctx, ENCHIP_ERR_ARG, "attention_bias: %lld query blocks of %d heads are more than one launch holds",
                    (long long)per, p.heads);
    const int64_t chunk = most / per, nseq = p.nseq;
    for (int64_t z0 = 0; z0 < nseq; z0 += chunk) {
        const int64_t nz = std::min(chunk, nseq - z0), row = z0 * p.L;
        enchip::AttnBias c = p;
        c.q += row * p.ldq, c.k += row * p.ldk, c.v += row * p.ldv, c.out += row * p.ldo;
        c.nseq = (int)nz;
        hipLaunchKernelGGL(fn, dim3((unsigned)(per * nz * sets)), dim3((unsigned)threads), (size_t)lds, s, c);
    }
    return check_launch(ctx, "attention_bias");
}

// Heads of one key head that a workgroup of nw wavefronts takes beside each other: a power of two of them, its log2.
int heads_beside(int64_t group, int nw) {
    int share = 0;
    while (share < 3 && (2 << share) <= nw && (group >> share) % 2 == 0) ++share;
    return share;
}

// p's spans longest first, in scratch, for query blocks of 2^qs rows.
int order_spans(enchip_ctx *ctx, enchip::AttnBias &p, int qs, hipStream_t s) {
    int rc;
    if ((rc = ensure(ctx, &ctx->d_att, &ctx->att_cap, (size_t)p.nseq * sizeof(int4)))) return rc;
    if ((rc = scratch_wait(ctx, s))) return rc;
    int4 *list = reinterpret_cast<int4 *>(ctx->d_att);
    hipLaunchKernelGGL(enchip::attention_bias_order, dim3(1), dim3(enchip::AB_ORDER_NT), 0, s, p.spans, p.nseq, p.L, qs, list);
    p.order = list;
    return check_launch(ctx, "attention_bias_order");
}

template <int HD, int NW, int QPW>
int attention_bias_tiles(enchip_ctx *ctx, enchip::AttnBias p, bool vec, int parts, bool order, hipStream_t s) {
    const int qs = __builtin_ctz(32 * NW * QPW), threads = 64 * NW, lds = enchip::AbLayout<HD, NW, QPW>::BYTES;
    p.share = heads_beside(p.group, NW);
    int rc;
    if (order) {
        if ((rc = order_spans(ctx, p, qs - p.share, s))) return rc;
        if ((rc = launch_attention_bias(ctx, vec ? enchip::attention_bias<HD, NW, QPW, true> : enchip::attention_bias<HD, NW, QPW, false>,
                                        lds, threads, qs - p.share, p, s)))
            return rc;
        return scratch_record(ctx, s);
    }
    if (parts == 1)
        return launch_attention_bias(ctx, vec ? enchip::attention_bias<HD, NW, QPW, true> : enchip::attention_bias<HD, NW, QPW, false>,
                                     lds, threads, qs - p.share, p, s);
    const size_t outputs = (size_t)parts * (size_t)p.rows * (size_t)p.heads;
    if ((rc = ensure(ctx, &ctx->d_att, &ctx->att_cap, outputs * (HD + 2) * sizeof(float)))) return rc;
    if ((rc = scratch_wait(ctx, s))) return rc;
    p.parts = parts;
    p.part = ctx->d_att;
    p.stat = ctx->d_att + outputs * HD;
    if ((rc = launch_attention_bias(ctx, enchip::attention_bias<HD, NW, QPW, true>, lds, threads, qs - p.share, p, s))) return rc;
    const int64_t per = p.spans ? p.L / 32 + p.nseq : (int64_t)((p.L + 31) / 32) * p.nseq;
    hipLaunchKernelGGL(enchip::attention_bias_join<HD>, dim3((unsigned)(per * p.heads)), dim3(256), 0, s, p);
    if ((rc = check_launch(ctx, "attention_bias_join"))) return rc;
    return scratch_record(ctx, s);
}

template <int HD, int NW>
int attention_bias_split(enchip_ctx *ctx, enchip::AttnBias p, bool order, hipStream_t s) {
    if (!order) return launch_attention_bias(ctx, enchip::attention_bias_split<HD, NW>, enchip::AbSplit<HD, NW>::BYTES, 64 * NW, 5, p, s);
    int rc;
    if ((rc = order_spans(ctx, p, 5, s))) return rc;
    if ((rc = launch_attention_bias(ctx, enchip::attention_bias_split<HD, NW>, enchip::AbSplit<HD, NW>::BYTES, 64 * NW, 5, p, s))) return rc;
    return scratch_record(ctx, s);
}

// How an attention runs, from its sizes (spans: as if all had their mean length).
//   split  attention_bias_split, while a workgroup per 32 queries leaves CUs for 1.5 rounds and no head has more
//          than 512 keys. Measured on MI355X, 12 heads of 64, us, split against tiles: 1 x 512 rows 12.9 against 23,
//          4 x 128 6.3 against 11.5; past the rule 4 x 512 34 against 31, 1 x 768 29.4 against 28.5.
//   else by tiles, the form (heads of 64: 512 queries a workgroup, or 256 and two workgroups a CU) and the parts that
//   the keys are split into with the least estimated time. Measured for w workgroups on a CU, us per 64-key tile:
//          heads of 32   1.9 alone, 3.1 for two at once      heads of 64, 256 queries   3.65, 5.0
//          heads of 128  4.6, one at once                    heads of 64, 512 queries   4.4, one at once
//   and 8 for each round's first loads and stores; joining parts 6 + 1.5 a part, and their bytes at 4 TB/s. With it
//   (12 heads of 64): 1 x 8192 rows 637 by 256 queries, 560 by 512, 546 in four parts; 1 x 2048 138 -> 58 in five;
//   1 x 1024 60 -> 34; 24 x 512 95 by 512, 85 by 256; 20011 packed rows of 1 to 1024 194 by 512, 152 by 256.
//   Rows of 64 and less whose heads of 128 do not share keys four and more: attention_bias_split with a wavefront alone
//   (1000 x 16 rows 118 -> 37, 200 x 64 41 -> 34, 5000 packed rows of 1 to 64 50 -> 22; 64 x 128 29.5 against 32).
//   Spans go longest first (attention_bias_order, a launch of 5 us) where a workgroup and a half a CU may come of
//   them: 20011 rows of documents of 1 to 1024, 12 heads of 64 154 -> 130, 16 heads of 128 316 -> 295, 5000 of them 97 -> 74;
//   64 x 512 padded rows 162 -> 75 (as they come, the padding's query blocks are a workgroup each); 64 equal spans of
//   512 270 -> 179, 16 heads of 128 that share 4 key heads 457 -> 460. 2500 rows, under the rule, 35.8 -> 36.6.
//   For a wavefront alone where the mean is past 32 rows and 8 wavefronts a CU may come of them: 20011 rows of 1 to 400 12
//   heads of 64 109 -> 100, 8 heads of 128 179 -> 147, of 1 to 200 77 -> 76 and 126 -> 115; 5000 rows of 1 to 64 21.6 -> 24.
struct AttnPlan {
    int split;  // wavefronts of attention_bias_split, 0: tiles
    bool wide;
    int parts;
    bool order;  // spans longest first
};

AttnPlan attention_plan(const enchip_ctx *ctx, const enchip::AttnBias &p, int64_t hd) {
    AttnPlan plan{0, false, 1, false};
    const int64_t cus = ctx->num_cus, len = p.spans ? std::max<int64_t>(1, p.L / p.nseq) : p.L;
    auto blocks = [&](int64_t rows, int64_t heads) { return (len + rows - 1) / rows * p.nseq * heads; };
    if (len <= 512 && 2 * blocks(32, p.heads) <= 3 * cus) plan.split = 8;
    else if (len <= 64 && (hd < 128 || heads_beside(p.group, 8) < 2)) plan.split = 1;
    // blocks of 32 rows, of all heads; below single any form's rounded grid is one launch
    const int64_t join = (p.spans ? p.L / 32 + p.nseq : (int64_t)((p.L + 31) / 32) * p.nseq) * p.heads, single = (int64_t)1 << 22;
    const bool sorts = p.spans != nullptr && p.nseq > 1 && p.nseq <= enchip::AB_ORDER_MAX && join < single;
    if (plan.split == 1) plan.order = sorts && len > 32 && join >= 8 * cus;
    if (plan.split) return plan;
    const int64_t tiles = (len + enchip::FA_KT - 1) / enchip::FA_KT;
    // with parts one launch holds all: the join's 256 threads for 32 rows, the tiles' 512 for 256 and each of 8 parts
    const int most = join < single ? (int)std::min<int64_t>(8, tiles) : 1;
    double least = 0.0;
    for (int wide = 0; wide <= (hd == 64 ? 1 : 0); ++wide) {
        const bool two = hd == 32 || (hd == 64 && !wide);  // workgroups at once on a CU
        const double alone = hd == 32 ? 1.9 : hd == 128 ? 4.6 : wide ? 4.4 : 3.65, both = hd == 32 ? 3.1 : 5.0;
        const int share = heads_beside(p.group, hd == 64 && !wide ? 4 : 8);
        const int64_t n = blocks((wide ? 512 : 256) >> share, p.heads >> share);
        for (int parts = 1; parts <= most; ++parts) {
            const int64_t w = (n * parts + cus - 1) / cus, rounds = two ? (w + 1) / 2 : w;
            const double tile = two ? (double)(w / 2) * both + (double)(w % 2) * alone : (double)w * alone;
            double us = (double)((tiles + parts - 1) / parts) * tile + 8.0 * (double)rounds;
            if (parts > 1) us += 6.0 + 1.5 * parts + 8.0 * parts * (double)p.rows * p.heads * (double)hd / 4e6;
            if (least == 0.0 || us < least) {
                least = us;
                plan.wide = wide != 0;
                plan.parts = parts;
            }
        }
    }
    const int share = heads_beside(p.group, hd == 64 && !plan.wide ? 4 : 8);
    const int64_t n = (p.L / ((plan.wide ? 512 : 256) >> share) + p.nseq) * (p.heads >> share);
    plan.order = sorts && plan.parts == 1 && 2 * n >= 3 * cus;
    return plan;
}

}  // namespace

extern "C" {

int enchip_attention_bias_dev(enchip_ctx *ctx, enchip_relpos relpos, const float *d_q, int64_t ldq, const float *d_k, int64_t ldk,
                              const float *d_v, int64_t ldv, float *d_out, int64_t ldo, const int32_t *d_spans, int64_t nseq,
                              int64_t L, int64_t heads, int64_t kv_heads, int64_t head_dim, float scale, void *stream) {
    if (!ctx) return ENCHIP_ERR_ARG;
    std::lock_guard<std::mutex> g(ctx->mu);
    RelPos r;
    if (relpos != 0) {
        auto it = ctx->relpos.find(relpos);
        if (it == ctx->relpos.end()) return fail(ctx, ENCHIP_ERR_HANDLE, "unknown relpos handle %llu", (unsigned long long)relpos);
        r = it->second;
    }
    if (head_dim != 32 && head_dim != 64 && head_dim != 128)
        return fail(ctx, ENCHIP_ERR_ARG, "attention_bias: head_dim must be 32, 64 or 128, got %lld", (long long)head_dim);
    const int64_t max_ld = INT32_MAX / enchip::FA_KT;
    if (nseq < 0 || L < 0 || L > ((int64_t)1 << 30) || heads < 0 || heads > 65535 || kv_heads < 0 || (heads > 0 && kv_heads < 1) ||
        (kv_heads > 0 && heads % kv_heads != 0) || nseq > (d_spans ? (int64_t)1 << 22 : (int64_t)INT32_MAX) ||
        (!d_spans && nseq * L > ((int64_t)1 << 31)) || ldq < heads * head_dim || ldo < heads * head_dim ||
        ldk < kv_heads * head_dim || ldv < kv_heads * head_dim || ldq % 4 || ldk % 4 || ldv % 4 || ldq > max_ld || ldk > max_ld ||
        ldv > max_ld)
        return fail(ctx, ENCHIP_ERR_ARG,
                    "attention_bias: bad shape nseq=%lld L=%lld heads=%lld kv_heads=%lld ldq=%lld ldk=%lld ldv=%lld ldo=%lld "
                    "(kv_heads dividing heads; ldq, ldk, ldv multiples of 4 covering the heads, below 2^25)",
                    (long long)nseq, (long long)L, (long long)heads, (long long)kv_heads, (long long)ldq, (long long)ldk,
                    (long long)ldv, (long long)ldo);
    if (relpos != 0 && r.heads != heads)
        return fail(ctx, ENCHIP_ERR_ARG, "attention_bias: a bias of %lld heads for %lld", (long long)r.heads, (long long)heads);
    if (nseq == 0 || L == 0 || heads == 0) return ENCHIP_OK;
    if (!d_q || !d_k || !d_v || !d_out) return fail(ctx, ENCHIP_ERR_ARG, "attention_bias: null pointer");
    if ((uintptr_t)d_q % 16 || (uintptr_t)d_k % 16 || (uintptr_t)d_v % 16 || (uintptr_t)d_spans % 8)
        return fail(ctx, ENCHIP_ERR_ARG, "attention_bias: q, k and v must be 16-byte aligned, spans 8-byte aligned");
    HIP_TRY(ctx, hipSetDevice(ctx->device));
    hipStream_t s = stream ? (hipStream_t)stream : ctx->stream;
    enchip::AttnBias p;
    p.q = d_q, p.k = d_k, p.v = d_v, p.out = d_out;
    p.ldq = ldq, p.ldk = ldk, p.ldv = ldv, p.ldo = ldo;
    p.spans = reinterpret_cast<const int2 *>(d_spans);
    p.table = r.d_table;
    p.nseq = (int)nseq, p.heads = (int)heads, p.group = (int)(heads / kv_heads), p.reach = (int)r.reach;
    p.L = (int)L;
    p.scale = scale;
    p.share = 0;
    p.block0 = 0;
    p.parts = 1;
    p.part = p.stat = nullptr;
    p.order = nullptr;
    p.rows = d_spans ? L : nseq * L;
    const bool vec = ldo % 4 == 0 && (uintptr_t)d_out % 16 == 0;
    const AttnPlan plan = attention_plan(ctx, p, head_dim);
    if (plan.split == 8 && head_dim == 32) return attention_bias_split<32, 8>(ctx, p, plan.order, s);
    if (plan.split == 8 && head_dim == 64) return attention_bias_split<64, 8>(ctx, p, plan.order, s);
    if (plan.split == 8) return attention_bias_split<128, 8>(ctx, p, plan.order, s);
    if (plan.split == 1 && head_dim == 32) return attention_bias_split<32, 1>(ctx, p, plan.order, s);
    if (plan.split == 1 && head_dim == 64) return attention_bias_split<64, 1>(ctx, p, plan.order, s);
    if (plan.split == 1) return attention_bias_split<128, 1>(ctx, p, plan.order, s);
    if (head_dim == 32) return attention_bias_tiles<32, 8, 1>(ctx, p, vec, plan.parts, plan.order, s);
    if (head_dim == 64 && plan.wide) return attention_bias_tiles<64, 8, 2>(ctx, p, vec, plan.parts, plan.order, s);
    if (head_dim == 64) return attention_bias_tiles<64, 4, 2>(ctx, p, vec, plan.parts, plan.order, s);
    return attention_bias_tiles<128, 8, 1>(ctx, p, vec, plan.parts, plan.order, s);
}

// ---------------------------------------------------------------------------- low-rank adapters

}  // extern "C"

namespace {

constexpr int64_t kMaxAdapterBytes = (int64_t)1 << 36;

int find_adapters(enchip_ctx *c, enchip_adapters h, AdapterSet **out) {
    auto it = c->adapters.find(h);
    if (it == c->adapters.end()) return fail(c, ENCHIP_ERR_HANDLE, "unknown adapters handle %llu", (unsigned long long)h);
    *out = &it->second;
    return ENCHIP_OK;
}

int64_t a_bytes(const AdapterSet &s) { return s.kb * s.rt * 3 * 1024; }  // of a slot
int64_t b_bytes(const AdapterSet &s) { return s.nb * s.rt * 3 * 1024; }
int64_t f_floats(const AdapterSet &s) { return 16 * s.rt * round_up(s.K, 4); }

void free_adapters(const AdapterSet &s) {
    (void)hipFree(s.d_a);
    (void)hipFree(s.d_b);
    (void)hipFree(s.d_f);
    (void)hipFree(s.d_up);
}

enchip::Adapters view(const enchip_ctx *c, const AdapterSet &set, const int32_t *d_ids) {
    enchip::Adapters p;
    p.a = reinterpret_cast<const enchip::bf16x8 *>(set.d_a);
    p.b = reinterpret_cast<const enchip::bf16x8 *>(set.d_b);
    p.af = set.d_f;
    p.t = reinterpret_cast<enchip::bf16x8 *>(c->d_low);
    p.ids = d_ids;
    p.slots = (int)set.slots, p.kb = (int)set.kb, p.nb = (int)set.nb, p.rt = (int)set.rt;
    return p;
}

int ensure_low(enchip_ctx *c, const AdapterSet &set, int64_t M) {
    return ensure(c, &c->d_low, &c->low_cap, (size_t)((M + 31) / 32 * set.rt * 3 * 1024));
}

constexpr int64_t kHeldK = 4096;  // widest rows that adapter_down quantizes

// The rows' low-rank parts into scratch, and with q their codes (ldq the weight's padded K, at most kHeldK).
// Few rows leave CUs idle: their rank tiles go to workgroups of their own.
int launch_down(enchip_ctx *c, const enchip::Adapters &p, const float *d_a, int64_t lda, int64_t M, int64_t K, const enchip::RowCodes *q,
                hipStream_t s) {
    const bool vec = lda % 4 == 0 && K % 4 == 0 && (uintptr_t)d_a % 16 == 0;
    const int64_t blocks = (M + 15) / 16, apart = std::max<int64_t>(1, 2 * c->num_cus / blocks);
    const bool four = p.rt > 1 && apart < p.rt;  // rank tiles four at a time
    // a workgroup a CU or less: 16 wavefronts, half as many steps each (1500 rows, K = 1000: 7.6 us -> 7.0)
    const bool few = blocks <= c->num_cus;
    const dim3 grid((unsigned)blocks, (unsigned)(four ? std::min<int64_t>(apart, (p.rt + 3) / 4) : p.rt));
    const enchip::RowCodes codes = q ? *q : enchip::RowCodes{};
#define AD_DOWN(V, C, NW, KBW)                                                                                                       \
    do {                                                                                                                             \
        if (four) hipLaunchKernelGGL((enchip::adapter_down<V, C, NW, KBW, 4>), grid, dim3(64 * NW), 0, s, d_a, lda, M, (int)K, p, codes); \
        else hipLaunchKernelGGL((enchip::adapter_down<V, C, NW, KBW, 1>), grid, dim3(64 * NW), 0, s, d_a, lda, M, (int)K, p, codes); \
    } while (0)
#define AD_K(V)                                                  \
    do {                                                         \
        if (!q && few) AD_DOWN(V, false, 16, 2);                 \
        else if (!q) AD_DOWN(V, false, 8, 4);                    \
        else if (q->ldq <= 256) AD_DOWN(V, true, 8, 1);          \
        else if (few && q->ldq <= 512) AD_DOWN(V, true, 16, 1);  \
        else if (few && q->ldq <= 1024) AD_DOWN(V, true, 16, 2); \
        else if (q->ldq <= 512) AD_DOWN(V, true, 8, 2);          \
        else if (q->ldq <= 1024) AD_DOWN(V, true, 8, 4);         \
        else if (q->ldq <= 2048) AD_DOWN(V, true, 16, 4);        \
        else AD_DOWN(V, true, 16, 8);                            \
    } while (0)
    if (vec) AD_K(true);
    else AD_K(false);
#undef AD_K
#undef AD_DOWN
    return check_launch(c, "adapter_down");
}

// dst = y + adapters, chunk after chunk of rows (32-bit thread numbers of a launch). Arguments checked.
int run_adapters(enchip_ctx *c, const AdapterSet &set, const float *d_a, int64_t lda, int64_t M, const int32_t *d_ids,
                 const float *d_y, int64_t ldy, float *d_dst, int64_t ldd, hipStream_t s) {
    const int64_t panels = (set.N + 127) / 128;
    const int64_t chunk = std::min(kRowChunk, std::max<int64_t>(1, ((int64_t)1 << 23) / panels) * 32);
    int rc;
    if ((rc = ensure_low(c, set, std::min(M, chunk)))) return rc;
    if ((rc = scratch_wait(c, s))) return rc;
    for (int64_t r0 = 0; r0 < M; r0 += chunk) {
        const int64_t n = std::min(chunk, M - r0);
        const enchip::Adapters p = view(c, set, d_ids + r0);
        if ((rc = launch_down(c, p, d_a + r0 * lda, lda, n, set.K, nullptr, s))) return rc;
        hipLaunchKernelGGL(enchip::adapter_up, dim3((unsigned)((n + 31) / 32 * panels)), dim3(256), 0, s, d_y + r0 * ldy, ldy,
                           d_dst + r0 * ldd, ldd, n, (int)set.N, p, (int)panels);
    }
    if ((rc = check_launch(c, "adapter_up"))) return rc;
    return scratch_record(c, s);
}

// The W8A8 product of quantized rows with their adapters, on the kernels of enchip_w8a8_linear_dev (few rows:
// row-major codes; else fragment-major, in pieces or gemm_w8a8_pt's tiles). M fits one launch.
template <int EPI>
void launch_linear(enchip_ctx *c, const Weight &w, const int8_t *aq, const float *as, const float *bias, float *out, int64_t M,
                   const enchip::Adapters &p, hipStream_t s) {
    using namespace enchip;
    const int m = (int)M, n = (int)w.N, kp = (int)w.Kp;
    if (M <= c->small_m) {
        const dim3 grid((unsigned)((w.N + 31) / 32), (unsigned)((M + GV_ROWS - 1) / GV_ROWS)), block(64 * GV_WAVES);
        const int64_t per_wave = (w.Kp / 32 + GV_WAVES - 1) / GV_WAVES;
#define GV_LAUNCH(NB) \
    hipLaunchKernelGGL((gemv_w8a8_adapters<EPI, NB>), grid, block, 0, s, aq, w.Kp, w.d_w, as, w.d_s, bias, out, w.N, m, n, kp, p)
        if (per_wave <= 1) GV_LAUNCH(1);
        else if (per_wave == 2) GV_LAUNCH(2);
        else if (per_wave <= 4) GV_LAUNCH(4);
        else GV_LAUNCH(8);
#undef GV_LAUNCH
        return;
    }
    const bool pt = use_persistent(w, aq, w.Kp, out, w.N, M, true);
    const int f = piece_form(c, w, M, EPI, !pt);
    if (pt && f < 0) {
        // 64-row tiles at any M: with the adapters' sums 128-row ones spill (32768 x 1024, K = 1024, rank 16: 63 us
        // against 57; without adapters 47)
        const int tn = (int)((w.N + PT_BN - 1) / PT_BN), tiles = (int)((M + PT_BM_SMALL - 1) / PT_BM_SMALL) * tn;
        const dim3 grid((unsigned)persistent_grid(c, tiles)), block(64 * PT_NW);
        if (pt_prio(w, EPI))
            hipLaunchKernelGGL((gemm_w8a8_pt_adapters<PT_BM_SMALL, PT_BN, PT_BK, PT_PW, EPI, PT_NW, 1, Adapters>), grid, block, 0, s, aq,
                               w.Kp, w.d_w, as, w.d_s, bias, out, w.N, m, n, kp, tn, tiles, p);
        else
            hipLaunchKernelGGL((gemm_w8a8_pt_adapters<PT_BM_SMALL, PT_BN, PT_BK, PT_PW, EPI, PT_NW, 0, Adapters>), grid, block, 0, s, aq,
                               w.Kp, w.d_w, as, w.d_s, bias, out, w.N, m, n, kp, tn, tiles, p);
        return;
    }
#define PIECE(F, VEC)                                                                                                            \
    do {                                                                                                                         \
        constexpr int CM = kPieces[F].cm, CN = kPieces[F].cn;                                                                    \
        const int64_t pn = (w.N + CN - 1) / CN;                                                                                  \
        hipLaunchKernelGGL((gemm_w8a8_adapters<CM, CN, EPI, PT_NW, PT_PW, VEC, Adapters>), dim3((unsigned)((M + CM - 1) / CM * pn)), \
                           dim3(64 * PT_NW), 0, s, aq, w.d_w, as, w.d_s, bias, out, w.N, m, n, kp, (int)pn, p);                  \
    } while (0)
    const bool vec = w.N % 4 == 0 && (uintptr_t)out % 16 == 0;
    if (f == 0 && vec) PIECE(0, true);
    else if (f == 0) PIECE(0, false);
    else if (f == 1 && vec) PIECE(1, true);
    else if (f == 1) PIECE(1, false);
    else if (vec) PIECE(2, true);
    else PIECE(2, false);
#undef PIECE
}

// Few rows in one launch (gemv_w8a8_q_adapters): every workgroup of 32 columns quantizes its 8 rows and forms their
// low-rank parts again, so A is small (its 16 rt rows of a slot, once a row a workgroup) and the launch about two
// workgroups a CU at rt = 1. LDS stays under 64 KiB. One launch against two, us, every row another adapter of 32
// (all rows one adapter's):
//   16 rows, K = 384, N = 1536, rank 8    6.0 against 22.4 (5.8 against 11.1)
//   16 rows, K = 768, N = 768, rank 32    10.8 against 29.2 (10.7 against 13.8)
//   32 rows, K = 768, N = 2304, rank 16 (288 workgroups)     12.8 against 29.5 (12.4 against 14.0)
//   32 rows, K = 1024, N = 4096, rank 16 (512 workgroups)    19.1 against 38.2 (17.6 against 15.0)
// and past it two: 32 rows, K = 768, N = 2304, rank 32 36.5 (15.0), K = 1024, N = 4096, rank 32 45.4 (16.0), where one took
// 19.0 and 27.2 with 8 adapters. Two would win only where most rows share an adapter, which the host does not know.
bool one_launch(const enchip_ctx *c, const Weight &w, const AdapterSet &set, int64_t M, const float *d_a) {
    const int64_t groups = (w.N + 31) / 32 * ((M + enchip::GVQ_ROWS - 1) / enchip::GVQ_ROWS);
    return M <= c->small_m && M <= 32 && w.K <= 1024 && w.K % 4 == 0 && (uintptr_t)d_a % 16 == 0 &&
           16 * set.rt <= enchip::Adapters::ROW_RANKS && groups * set.rt <= 2 * (int64_t)c->num_cus;
}

template <int EPI>
int launch_one(enchip_ctx *c, const Weight &w, const enchip::Adapters &p, const float *d_a, int64_t M, const float *bias, float *out,
               hipStream_t s) {
    using namespace enchip;
    const dim3 grid((unsigned)((w.N + 31) / 32), (unsigned)((M + GVQ_ROWS - 1) / GVQ_ROWS));
    const size_t lds = (size_t)gvq_lds_bytes((int)w.Kp);
#define GVQ_LAUNCH(QCH)                                                                                                     \
    hipLaunchKernelGGL((gemv_w8a8_q_adapters<EPI, QCH>), grid, dim3(64 * GVQ_WAVES), lds, s, d_a, w.d_w, w.d_s, bias, out, w.N, (int)M, \
                       (int)w.N, (int)w.K, (int)w.Kp, p)
    if (w.K <= 256) GVQ_LAUNCH(1);
    else if (w.K <= 512) GVQ_LAUNCH(2);
    else if (w.K <= 768) GVQ_LAUNCH(3);
    else GVQ_LAUNCH(4);
#undef GVQ_LAUNCH
    return check_launch(c, "gemv_w8a8_q_adapters");
}

// act(W8A8(a) + bias + adapters): the rows quantized and their low-rank parts formed in one pass over them, then
// the product with the adapters in its epilogue. Chunk after chunk of rows, for which gemm_w8a8_pt's byte offsets
// and a launch's thread numbers fit 32 bits. Arguments checked.
int run_linear_adapters(enchip_ctx *c, const Weight &w, const AdapterSet &set, const float *d_a, int64_t M, const int32_t *d_ids,
                        const float *d_bias, int act, float *d_dst, hipStream_t s) {
    if (one_launch(c, w, set, M, d_a)) {  // no scratch
        const enchip::Adapters p = view(c, set, d_ids);
        return act == ENCHIP_ACT_GELU ? launch_one<enchip::EPI_F32_GELU>(c, w, p, d_a, M, d_bias, d_dst, s)
                                      : launch_one<enchip::EPI_F32>(c, w, p, d_a, M, d_bias, d_dst, s);
    }
    const int64_t by_codes = (((int64_t)1 << 31) - 1) / w.Kp, by_pieces = ((int64_t)1 << 34) / round_up(w.N, 32);
    const int64_t chunk = M <= c->small_m ? M : std::max<int64_t>(128, std::min({kRowChunk, by_codes, by_pieces}) / 128 * 128);
    int rc;
    if ((rc = ensure_act_scratch(c, std::min(M, chunk), w.Kp))) return rc;
    if ((rc = ensure_low(c, set, std::min(M, chunk)))) return rc;
    if ((rc = scratch_wait(c, s))) return rc;
    for (int64_t r0 = 0; r0 < M; r0 += chunk) {
        const int64_t n = std::min(chunk, M - r0);
        const enchip::Adapters p = view(c, set, d_ids + r0);
        const float *a = d_a + r0 * w.K;
        const bool frag = n > c->small_m;
        const enchip::RowCodes q{c->d_aq, c->d_as, w.Kp, frag};
        if (w.Kp > kHeldK && (rc = launch_quant(c, a, n, w.K, c->d_aq, w.Kp, c->d_as, s, frag))) return rc;
        if ((rc = launch_down(c, p, a, w.K, n, w.K, w.Kp > kHeldK ? nullptr : &q, s))) return rc;
        if (act == ENCHIP_ACT_GELU) launch_linear<enchip::EPI_F32_GELU>(c, w, c->d_aq, c->d_as, d_bias, d_dst + r0 * w.N, n, p, s);
        else launch_linear<enchip::EPI_F32>(c, w, c->d_aq, c->d_as, d_bias, d_dst + r0 * w.N, n, p, s);
        if ((rc = check_launch(c, "linear_adapters"))) return rc;
    }
    return scratch_record(c, s);
}

}  // namespace

extern "C" {

int enchip_adapters_create(enchip_ctx *ctx, int64_t K, int64_t N, int64_t rank, int64_t slots, enchip_adapters *out) {
    if (!ctx) return ENCHIP_ERR_ARG;
    std::lock_guard<std::mutex> g(ctx->mu);
    if (!out) return fail(ctx, ENCHIP_ERR_ARG, "adapters_create: out is NULL");
    *out = 0;
    if (K < 1 || K > kMaxK || N < 1 || N > ((int64_t)1 << 24) || rank < 1 || rank > 256 || slots < 1 || slots > 65536)
        return fail(ctx, ENCHIP_ERR_ARG, "adapters_create: bad shape K=%lld N=%lld rank=%lld slots=%lld", (long long)K, (long long)N,
                    (long long)rank, (long long)slots);
    AdapterSet set;
    set.K = K, set.N = N, set.rank = rank, set.slots = slots;
    set.kb = (K + 31) / 32, set.nb = round_up(N, 256) / 32, set.rt = (rank + 15) / 16;
    // a block of A is 32 k x 16 ranks, one of B 32 columns x 16 ranks: 1 KiB a part each
    const int64_t bytes[4] = {slots * a_bytes(set), slots * b_bytes(set), slots * f_floats(set) * 4, rank * (K + N) * 4};
    if (bytes[0] + bytes[1] + bytes[2] > kMaxAdapterBytes)
        return fail(ctx, ENCHIP_ERR_ARG, "adapters_create: %lld slots of K=%lld N=%lld rank=%lld are past 2^36 bytes", (long long)slots,
                    (long long)K, (long long)N, (long long)rank);
    HIP_TRY(ctx, hipSetDevice(ctx->device));
    size_t cap[4] = {};
    int rc = ensure(ctx, &set.d_a, &cap[0], (size_t)bytes[0], false);
    if (!rc) rc = ensure(ctx, &set.d_b, &cap[1], (size_t)bytes[1], false);
    if (!rc) rc = ensure(ctx, &set.d_f, &cap[2], (size_t)bytes[2], false);
    if (!rc) rc = ensure(ctx, &set.d_up, &cap[3], (size_t)bytes[3], false);
    if (!rc) {
        hipError_t e = hipMemsetAsync(set.d_a, 0, (size_t)bytes[0], ctx->stream);
        if (e == hipSuccess) e = hipMemsetAsync(set.d_b, 0, (size_t)bytes[1], ctx->stream);
        if (e == hipSuccess) e = hipMemsetAsync(set.d_f, 0, (size_t)bytes[2], ctx->stream);
        if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
        if (e != hipSuccess) rc = fail(ctx, ENCHIP_ERR_HIP, "adapters_create: %s", hipGetErrorString(e));
    }
    if (!rc) {
        try {
            ctx->adapters[ctx->next_handle] = set;
        } catch (const std::bad_alloc &) {
            rc = fail(ctx, ENCHIP_ERR_OOM, "adapters_create: out of host memory");
        }
    }
    if (rc) {
        free_adapters(set);
        return rc;
    }
    *out = ctx->next_handle++;
    return ENCHIP_OK;
}

int enchip_adapters_set(enchip_ctx *ctx, enchip_adapters h, int64_t slot, const float *A, const float *B, float scale) {
    if (!ctx) return ENCHIP_ERR_ARG;
    std::lock_guard<std::mutex> g(ctx->mu);
    AdapterSet *set;
    int rc = find_adapters(ctx, h, &set);
    if (rc) return rc;
    if (slot < 0 || slot >= set->slots) return fail(ctx, ENCHIP_ERR_ARG, "adapters_set: slot %lld of %lld", (long long)slot, (long long)set->slots);
    if (!A || !B) return fail(ctx, ENCHIP_ERR_ARG, "adapters_set: null pointer");
    const int64_t K = set->K, N = set->N, R = set->rank;
    for (int64_t i = 0; i < R * K; ++i)
        if (!(std::fabs(A[i]) < 0x1p127f))
            return fail(ctx, ENCHIP_ERR_ARG, "adapters_set: A[%lld][%lld] is %g", (long long)(i / K), (long long)(i % K), (double)A[i]);
    for (int64_t i = 0; i < N * R; ++i)
        if (!(std::fabs((double)scale * (double)B[i]) < 0x1p127))
            return fail(ctx, ENCHIP_ERR_ARG, "adapters_set: scale %g times B[%lld][%lld] is %g", (double)scale, (long long)(i / R),
                        (long long)(i % R), (double)scale * (double)B[i]);
    HIP_TRY(ctx, hipSetDevice(ctx->device));
    HIP_TRY(ctx, hipStreamSynchronize(ctx->stream));
    HIP_TRY(ctx, hipMemcpy(set->d_up, A, (size_t)(R * K) * sizeof(float), hipMemcpyHostToDevice));
    HIP_TRY(ctx, hipMemcpy(set->d_up + R * K, B, (size_t)(N * R) * sizeof(float), hipMemcpyHostToDevice));
    const int64_t threads = (set->kb + set->nb) * set->rt * 64;
    hipLaunchKernelGGL(enchip::adapter_pack, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, ctx->stream, set->d_up, set->d_up + R * K,
                       (double)scale, (int)K, (int)N, (int)R, (int)set->kb, (int)set->nb, (int)set->rt,
                       reinterpret_cast<enchip::bf16x8 *>(set->d_a + slot * a_bytes(*set)),
                       reinterpret_cast<enchip::bf16x8 *>(set->d_b + slot * b_bytes(*set)), set->d_f + slot * f_floats(*set));
    if ((rc = check_launch(ctx, "adapter_pack"))) return rc;
    HIP_TRY(ctx, hipStreamSynchronize(ctx->stream));  // work on any stream finds the adapter whole
    return ENCHIP_OK;
}

int enchip_adapters_release(enchip_ctx *ctx, enchip_adapters h) {
    if (!ctx) return ENCHIP_ERR_ARG;
    std::lock_guard<std::mutex> g(ctx->mu);
    AdapterSet *set;
    int rc = find_adapters(ctx, h, &set);
    if (rc) return rc;
    HIP_TRY(ctx, hipSetDevice(ctx->device));
    HIP_TRY(ctx, hipStreamSynchronize(ctx->stream));
    free_adapters(*set);
    ctx->adapters.erase(h);
    return ENCHIP_OK;
}

int enchip_adapters_add_dev(enchip_ctx *ctx, enchip_adapters h, const float *d_a, int64_t lda, int64_t M, const int32_t *d_ids,
                            const float *d_y, int64_t ldy, float *d_dst, int64_t ldd, void *stream) {
    if (!ctx) return ENCHIP_ERR_ARG;
    std::lock_guard<std::mutex> g(ctx->mu);
    AdapterSet *set;
    int rc = find_adapters(ctx, h, &set);
    if (rc) return rc;
    if (M < 0 || M > ((int64_t)1 << 30) || lda < set->K || ldy < set->N || ldd < set->N)
        return fail(ctx, ENCHIP_ERR_ARG, "adapters_add: bad shape M=%lld lda=%lld ldy=%lld ldd=%lld for K=%lld N=%lld", (long long)M,
                    (long long)lda, (long long)ldy, (long long)ldd, (long long)set->K, (long long)set->N);
    if (d_y == d_dst && ldy != ldd)
        return fail(ctx, ENCHIP_ERR_ARG, "adapters_add: in place needs one pitch, not %lld and %lld", (long long)ldy, (long long)ldd);
    if (M == 0) return ENCHIP_OK;
    if (!d_a || !d_ids || !d_y || !d_dst) return fail(ctx, ENCHIP_ERR_ARG, "adapters_add: null pointer");
    HIP_TRY(ctx, hipSetDevice(ctx->device));
    hipStream_t s = stream ? (hipStream_t)stream : ctx->stream;
    return run_adapters(ctx, *set, d_a, lda, M, d_ids, d_y, ldy, d_dst, ldd, s);
}

int enchip_w8a8_linear_adapters_dev(enchip_ctx *ctx, enchip_weight hw, enchip_adapters h, const float *d_a, int64_t M,
                                    const int32_t *d_ids, const float *d_bias, int act, float *d_dst, void *stream) {
    if (!ctx) return ENCHIP_ERR_ARG;
    std::lock_guard<std::mutex> g(ctx->mu);
    Weight *w;
    AdapterSet *set;
    int rc = find_weight(ctx, hw, &w);
    if (rc || (rc = find_adapters(ctx, h, &set))) return rc;
    if (set->K != w->K || set->N != w->N)
        return fail(ctx, ENCHIP_ERR_ARG, "linear_adapters: adapters of K=%lld N=%lld for a weight of K=%lld N=%lld", (long long)set->K,
                    (long long)set->N, (long long)w->K, (long long)w->N);
    if (M < 0 || M > ((int64_t)1 << 30)) return fail(ctx, ENCHIP_ERR_ARG, "linear_adapters: bad M=%lld", (long long)M);
    if (act != ENCHIP_ACT_NONE && act != ENCHIP_ACT_GELU) return fail(ctx, ENCHIP_ERR_ARG, "linear_adapters: bad act %d", act);
    if (M == 0) return ENCHIP_OK;
    if (!d_a || !d_ids || !d_dst) return fail(ctx, ENCHIP_ERR_ARG, "linear_adapters: null pointer");
    HIP_TRY(ctx, hipSetDevice(ctx->device));
    hipStream_t s = stream ? (hipStream_t)stream : ctx->stream;
    return run_linear_adapters(ctx, *w, *set, d_a, M, d_ids, d_bias, act, d_dst, s);
}

}  // extern "C"

// context.h -- what the library's translation units share: the context, its errors, its growable scratch
// and the order of streams on it, and which kernels a W8A8 linear runs.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <mutex>
#include <new>
#include <string>
#include <unordered_map>
#include <utility>
#include <vector>

#include "enchip.h"
#include "gemm_persistent.h"
#include "kernels.h"

namespace enchip_host {


constexpr int64_t kMaxK = 131072;  // K*127*127 stays below 2^31: the int32 dot cannot wrap
constexpr int64_t kRowPad = 256;   // quantized-activation scratch rows are padded to this
constexpr int64_t kColPad = 256;   // weight output channels are padded to this

inline int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

struct Weight {
    int8_t *d_w = nullptr;  // fragment-major, [Np/32][Kp/32][1024]
    float *d_s = nullptr;   // [N]
    int64_t N = 0, K = 0, Np = 0, Kp = 0;
    bool inf_scale = false;  // some scale is +-inf: enchip_matmul_bt_q8 declines (see there)
};

// A weight of 4-bit codes and f16 group scales (enchip_weight4_register; weight_only.h).
struct Weight4 {
    int8_t *d_w = nullptr;    // [Np/64][Kp/32][64][16 B]
    uint16_t *d_s = nullptr;  // f16 [Np/64][G][64]
    int64_t N = 0, K = 0, group = 0, Np = 0, Kp = 0, G = 0;
};

// Rotary frequencies (enchip_rope_create).
struct Rope {
    double2 *d_turns = nullptr;  // [n] f_j / 2 pi less whole turns, in two parts
    int64_t n = 0;              // pairs
    float mscale = 1.0f;
};

// A learned bias by relative position (enchip_relpos_create).
struct RelPos {
    float *d_table = nullptr;  // [heads][2 reach + 1], times log2 e
    int64_t heads = 0, reach = 0;
};

// Low-rank adapters of one linear's shape (enchip_adapters_create; adapters.h).
struct AdapterSet {
    char *d_a = nullptr, *d_b = nullptr;  // the slots' parts
    float *d_f = nullptr;                 // A as it is
    float *d_up = nullptr;                // an adapter on its way in: A, then B
    int64_t K = 0, N = 0, rank = 0, slots = 0, kb = 0, nb = 0, rt = 0;
};

// The last failure this thread saw on a context (by its id), so that a thread reading
// enchip_last_error after its own failure gets its own message even when another
// thread has failed on the same context since.
struct ThreadError {
    uint64_t ctx_id = 0;
    std::string msg;
};
inline thread_local ThreadError g_thread_error;

}  // namespace enchip_host

struct enchip_ctx {
    uint64_t id = 0;  // unique per context for the life of the process
    int device = 0;
    hipStream_t stream = nullptr;
    int num_cus = 0, clock_khz = 0;
    std::string arch;
    std::mutex mu;
    std::string err = "no error";
    int8_t *noalloc = nullptr;  // this device's address of `scratch` (NULL: unavailable)
    std::string noalloc_err;
    std::unordered_map<uint64_t, enchip_host::Weight> weights;
    std::unordered_map<uint64_t, enchip_host::Weight4> weights4;  // handles of all kinds come from next_handle
    std::unordered_map<uint64_t, enchip_host::Rope> ropes;
    std::unordered_map<uint64_t, enchip_host::RelPos> relpos;
    std::unordered_map<uint64_t, enchip_host::AdapterSet> adapters;
    // Attention kernels whose dynamic-LDS limit has been raised on this context's device
    // (hipFuncSetAttribute, once per kernel and byte count rather than once per launch).
    std::vector<std::pair<const void *, size_t>> lds_set;
    uint64_t next_handle = 1;
    int64_t small_m = 32;
    int att_products = ENCHIP_ATT_FLASH_F16;  // enchip_set_attention_products
    // Device scratch (grown on demand, freed by enchip_close). Each growable buffer is
    // capped at scratch_limit bytes (enchip_set_scratch_limit; 0 = no cap).
    size_t scratch_limit = 0;
    // The last stream that enqueued work on the shared scratch (d_aq, d_as, d_cand) and
    // an event recorded after that work: a user on another stream waits for it first. Until the
    // first such user comes, work on the context's own stream records none.
    hipEvent_t scratch_ev = nullptr;
    hipStream_t scratch_stream = nullptr;
    bool scratch_pending = false, scratch_recorded = false, scratch_shared = false;
    // Set once work on the scratch has been captured into a graph, which keeps its addresses: buffers
    // that grow from then on are kept (retired) until enchip_close, not freed.
    bool scratch_captured = false;
    std::vector<void *> retired;
    int8_t *d_aq = nullptr;
    size_t aq_cap = 0;
    float *d_as = nullptr;
    size_t as_cap = 0;
    float *d_a = nullptr;
    size_t a_cap = 0;
    float *d_dst = nullptr;
    size_t dst_cap = 0;
    float *d_bias = nullptr;
    size_t bias_cap = 0;
    int32_t *d_acc = nullptr;
    size_t acc_cap = 0;
    float *d_fb = nullptr;  // enchip_matmul_bt_f32's b operand
    size_t fb_cap = 0;
    char *d_low = nullptr;  // the rows' low-rank parts (adapters.h)
    size_t low_cap = 0;
    float *d_att = nullptr;  // parts of an attention's contexts (attention_bias.h)
    size_t att_cap = 0;
    uint64_t *d_cand = nullptr;  // top-k candidates
    size_t cand_cap = 0;
    // enchip_ann_topk's device results, one block so that one copy brings them back:
    // hit indices (int32, M k), hit scores (f32, M k), then the fused route's list sizes
    // (uint32, M)
    int32_t *d_hits = nullptr;
    size_t hits_cap = 0;
    // enchip_ann_topk routing (enchip_ann_topk_stats)
    int64_t ann_fused_calls = 0, ann_fallbacks = 0;
    // Pinned host staging for the host entry points' large copies (kStageBytes). upload: two
    // slots of kStageChunk bytes, each fenced by an event recorded after its DMA. download: two
    // halves of kDownHalf bytes and, past them, the arrival words of copy_out's launches.
    char *h_stage = nullptr;
    hipEvent_t stage_ev[2] = {nullptr, nullptr};
    uint32_t down_epoch = 0;  // copy_out launches so far; 0 is no launch's word
};

namespace enchip_host {

inline int fail(enchip_ctx *c, int code, const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    c->err = buf;
    g_thread_error.ctx_id = c->id;
    g_thread_error.msg = buf;
    return code;
}

#define HIP_TRY(ctx, expr)                                                                  \
    do {                                                                                    \
        hipError_t e_ = (expr);                                                             \
        if (e_ != hipSuccess)                                                               \
            return fail((ctx), ENCHIP_ERR_HIP, "%s failed: %s", #expr, hipGetErrorString(e_)); \
    } while (0)

// Grows a device buffer to at least `bytes`. Contents are not preserved. Scratch
// buffers (not weights) are refused past the context's scratch limit, as a failed
// allocation would be.
template <typename T>
int ensure(enchip_ctx *c, T **p, size_t *cap, size_t bytes, bool scratch = true) {
    // checked before the capacity: a call that needs more than the cap declines even
    // when an earlier call already grew the buffer
    if (scratch && c->scratch_limit != 0 && bytes > c->scratch_limit)
        return fail(c, ENCHIP_ERR_OOM, "scratch of %zu bytes exceeds the context's scratch limit of %zu", bytes,
                    c->scratch_limit);
    if (bytes <= *cap && *p) return ENCHIP_OK;
    size_t want = std::max<size_t>(bytes, 256);
    if (*p && scratch && c->scratch_captured) {
        // grows at least twofold, so that all that is kept is less than what is in use
        want = std::max(want, c->scratch_limit ? std::min(2 * *cap, c->scratch_limit) : 2 * *cap);
        try {
            c->retired.push_back(*p);
        } catch (const std::bad_alloc &) {
            return fail(c, ENCHIP_ERR_OOM, "scratch: out of host memory");
        }
        *p = nullptr;
        *cap = 0;
    } else if (*p) {
        // the old buffer may still be read by work enqueued on another stream
        if (scratch && c->scratch_pending)
            (void)(c->scratch_recorded ? hipEventSynchronize(c->scratch_ev) : hipStreamSynchronize(c->stream));
        hipError_t e = hipFree(*p);
        *p = nullptr;
        *cap = 0;
        if (e != hipSuccess) return fail(c, ENCHIP_ERR_HIP, "hipFree: %s", hipGetErrorString(e));
    }
    hipError_t e = hipMalloc((void **)p, want);
    if (e != hipSuccess && want > std::max<size_t>(bytes, 256)) {
        (void)hipGetLastError();
        want = std::max<size_t>(bytes, 256);
        e = hipMalloc((void **)p, want);
    }
    if (e != hipSuccess) {
        *p = nullptr;
        (void)hipGetLastError();
        return fail(c, ENCHIP_ERR_OOM, "hipMalloc(%zu): %s", want, hipGetErrorString(e));
    }
    *cap = want;
    return ENCHIP_OK;
}

inline int check_launch(enchip_ctx *c, const char *what) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(c, ENCHIP_ERR_HIP, "launch %s: %s", what, hipGetErrorString(e));
    return ENCHIP_OK;
}

// A 1-D launch of `blocks` workgroups of `threads` must keep its global thread index
// below 2^32.
inline bool grid_fits(int64_t blocks, int64_t threads) {
    return blocks >= 0 && blocks * threads < ((int64_t)1 << 32);
}

// Rows per launch of the row kernels (at most 64 threads per row: 2^28 threads).
constexpr int64_t kRowChunk = (int64_t)1 << 22;

inline bool capturing(hipStream_t s) {
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    return hipStreamIsCapturing(s, &st) == hipSuccess && st != hipStreamCaptureStatusNone;
}

// Orders work about to use the shared scratch on stream s after the scratch's last
// user on another stream. Under stream capture the caller orders the streams (a
// captured graph cannot wait on an event recorded outside it).
inline int scratch_wait(enchip_ctx *c, hipStream_t s) {
    if (!c->scratch_pending || c->scratch_stream == s || capturing(s)) return ENCHIP_OK;
    hipError_t e;
    c->scratch_shared = true;
    if (!c->scratch_recorded) {  // the last user was the context's stream, alone so far
        if ((e = hipEventRecord(c->scratch_ev, c->stream)) != hipSuccess)
            return fail(c, ENCHIP_ERR_HIP, "hipEventRecord(scratch): %s", hipGetErrorString(e));
        c->scratch_recorded = true;
    }
    e = hipStreamWaitEvent(s, c->scratch_ev, 0);
    if (e != hipSuccess) return fail(c, ENCHIP_ERR_HIP, "hipStreamWaitEvent(scratch): %s", hipGetErrorString(e));
    return ENCHIP_OK;
}

// Marks the scratch as in use by the work just enqueued on stream s. An event costs the
// stream about 5 us on MI355X (a 512-row linear's two launches 12.7 us per call with it, 9.5
// without), so while no other stream has waited for the scratch, work on the context's own
// stream, which lives as long as the scratch and is captured by nobody, leaves it to the first
// that does (scratch_wait; that one waits for all the work enqueued there so far). From then on,
// and after work on a caller's stream, which may be gone by the next use, it is recorded here:
// another stream waits for the scratch's last use and for nothing after it.
inline int scratch_record(enchip_ctx *c, hipStream_t s) {
    const bool record = s != c->stream || c->scratch_shared;
    if (record) {
        if (s != c->stream && capturing(s)) {
            c->scratch_captured = true;
            return ENCHIP_OK;
        }
        hipError_t e = hipEventRecord(c->scratch_ev, s);
        if (e != hipSuccess) return fail(c, ENCHIP_ERR_HIP, "hipEventRecord(scratch): %s", hipGetErrorString(e));
    }
    c->scratch_recorded = record;
    c->scratch_stream = s;
    c->scratch_pending = true;
    return ENCHIP_OK;
}

// Ring depth of gemm_w8a8_pt: 2 stages, so the 64-deep K stages must be even (0 = not
// usable). A 3-stage ring speeds up the bare main loop by 2-9% on MI355X, but with the
// epilogue its register pressure spills and the whole kernel is no faster.
inline int pt_ring(const Weight &w) {
    return (w.Kp / enchip::PT_BK) % enchip::PT_PW == 0 ? enchip::PT_PW : 0;
}

// gemm_w8a8_pt's preconditions (gemm_persistent.h): a usable ring depth, 16-byte
// aligned A, 32-bit byte offsets into A and the weights, and 16-byte row-major output
// stores (N and the output pitch multiples of 4). Fragment-major A (af) has pitch Kp
// and is read up to the next multiple of PT_BM rows.
inline bool use_persistent(const Weight &w, const void *aq, int64_t lda, const void *out, int64_t ldo, int64_t M,
                    bool af) {
    const int64_t lim = (int64_t)1 << 31;
    const int64_t a_end = af ? round_up(M, enchip::PT_BM) * w.Kp : (M - 1) * lda + w.Kp;
    return pt_ring(w) != 0 && (lda % 16) == 0 && (!af || lda == w.Kp) && ((uintptr_t)aq % 16) == 0 &&
           a_end < lim && w.Np * w.Kp < lim && (w.N % 4) == 0 && (ldo % 4) == 0 && ((uintptr_t)out % 16) == 0;
}

// True when a GEMM on activations this library quantizes itself (into the context
// scratch, pitch Kp) runs gemm_w8a8_pt, which then takes them fragment-major.
inline bool route_af(const enchip_ctx *c, const Weight &w, int64_t M, const void *out, int64_t ldo) {
    return M > c->small_m && use_persistent(w, nullptr, w.Kp, out, ldo, M, true);
}

// gemm_pieces.h's piece size for a GEMM on fragment-major codes, as an index into kPieces
// (-1: gemm_w8a8_pt's or the general kernel's tiles). Pieces pay while their number is a few
// per CU; past that the larger tiles' fewer loads per output win. Measured on MI355X (graph
// replay; (M, N, K), 64 x 64 pieces' number, tiles -> pieces): bias only, (512, 4096, 1024),
// 512: 9.4 -> 8.6 us, (1024, 2304, 768), 576: 7.0 -> 7.6, (1024, 3072, 768), 768: 7.2 -> 8.7.
// With the GELU, whose VALU work the tiles leave to few wavefronts: (2048, 2304, 768), 1152:
// 15.1 -> 14.6 at 7% erf tails and 25.3 -> 16.4 at 25%, (2048, 3072, 768), 1536: 15.6 -> 18.3
// and 26.9 -> 20.1. `ragged`: the outputs gemm_w8a8_pt cannot store, against gemm_w8a8 on
// row-major codes (linears of N = 1001): (4000, K = 768), 1008 pieces, 22.0 -> 20.5 us, (5000,
// 384), 1264, 19.6 -> 21.0; with the GELU (5000, 768) 41.8 -> 28.3; (40, 768) 13.5 -> 6.0.
// Size: 32 x 32 while a CU gets few of them (long K: each wavefront's serial steps are what
// is left, and larger pieces load less), 64 x 32 for K <= 1024 or few pieces, else 64 x 64:
// (512, 768, 3072) 5.5 / 4.9 / 6.2 us, (1024, 768, 3072) 7.6 / 7.6 / 6.6, (512, 2304, 768)
// 5.5 / 5.5 / 6.1, (256, 768, 768) 2.9 / 3.3 / 4.2; with the GELU (1024, 768, 768)
// 5.4 / 6.2 / 6.9.
struct Piece {
    int cm, cn;
};
constexpr Piece kPieces[3] = {{32, 32}, {64, 32}, {64, 64}};

inline int piece_form(const enchip_ctx *c, const Weight &w, int64_t M, int epi, bool ragged) {
    const int64_t cus = c->num_cus;
    const bool gelu = epi == enchip::EPI_F32_GELU, short_k = w.Kp <= 1024;
    auto pieces = [&](int64_t cm, int64_t cn) { return ((M + cm - 1) / cm) * ((w.N + cn - 1) / cn); };
    if (pieces(64, 64) > (gelu ? 5 : ragged ? 4 : 2) * cus) return -1;
    if (pieces(32, 32) <= (gelu ? 2 : 1) * (short_k ? 2 : 1) * cus) return 0;
    return short_k || pieces(64, 32) <= (gelu ? 3 : 1) * cus ? 1 : 2;
}

inline int persistent_grid(const enchip_ctx *c, int64_t tiles, int per_cu = 2) {
    const int64_t full = std::max<int64_t>(8, ((int64_t)per_cu * c->num_cus) / 8 * 8);
    return (int)std::min<int64_t>(full, (tiles + 7) / 8 * 8);
}

// Tile height of gemm_w8a8_pt for M rows of a weight: 64-row tiles at 3 workgroups per CU
// when 128-row tiles would not fill the 2 per CU slots (small M), else 128. Measured on
// MI355X (K = 768, N = 3072, GELU): M = 4096 46 -> 35 us on config 2's pre-activations and
// 29 -> 25 us on an encoder's; at M = 32768 the 128-row tiles stay faster (164 against 166).
inline int pt_bm(const enchip_ctx *c, const Weight &w, int64_t M) {
    const int64_t tiles128 = ((M + enchip::PT_BM - 1) / enchip::PT_BM) * ((w.N + enchip::PT_BN - 1) / enchip::PT_BN);
    return tiles128 < 2 * (int64_t)c->num_cus ? enchip::PT_BM_SMALL : enchip::PT_BM;
}

// Main-loop wave priority of gemm_w8a8_pt for a weight and epilogue: raised for the
// bias-only epilogue when N or the padded K is at least 1024. Measured on MI355X (same
// process, interleaved): BERT-base QKV and FFN-down 4-10% faster, XLM-R-large QKV, O and
// FFN-down 6-9% faster; BERT-base O (768 x 768) 4% slower, so it keeps 0. The GELU
// epilogue keeps 0: raised, BERT-base FFN-up took 206 us per launch in the encode against
// 189 us (it ran 3-5% faster on uniformly random codes, whose pre-activations differ).
inline int pt_prio(const Weight &w, int epi) {
    return (epi == enchip::EPI_F32 || epi == enchip::EPI_TOPK) && (w.N >= 1024 || w.Kp >= 1024) ? 1 : 0;
}

inline int find_weight(enchip_ctx *c, enchip_weight h, Weight **out) {
    auto it = c->weights.find(h);
    if (it == c->weights.end()) return fail(c, ENCHIP_ERR_HANDLE, "unknown weight handle %llu", (unsigned long long)h);
    *out = &it->second;
    return ENCHIP_OK;
}

// Scratch for the quantized activations of M rows at pitch Kp.
inline int ensure_act_scratch(enchip_ctx *c, int64_t M, int64_t Kp) {
    const int64_t Mp = round_up(std::max<int64_t>(M, 1), kRowPad);
    int rc = ensure(c, &c->d_aq, &c->aq_cap, (size_t)(Mp * Kp));
    if (rc) return rc;
    return ensure(c, &c->d_as, &c->as_cap, (size_t)Mp * sizeof(float));
}

inline int act_code(int act) {
    return act == ENCHIP_ACT_GELU ? enchip::EPI_F32_GELU : enchip::EPI_F32;
}

inline enchip::FastDiv fast_div(int64_t d) {
    return {(uint32_t)d, d == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + (uint64_t)d - 1) / (uint64_t)d), d == 1 ? ~0u : 0u};
}

// Quantizes d_a[M,K] into q (zero-padded to ldq) and scale[M]: row-major q[M][ldq], or
// fragment-major (kernels.h frag_off) when frag. (enchip.hip)
int launch_quant(enchip_ctx *c, const float *d_a, int64_t M, int64_t K, int8_t *q, int64_t ldq, float *scale,
                 hipStream_t s, bool frag = false);

}  // namespace enchip_host

// The C entry points of the 8-bit key / value cache, the attention over it, the logits' rules and the draw: the checks of their arguments.
#include "backend.hpp"
#include "kv.hpp"
#include "logits.hpp"
#include "sample.hpp"

using namespace oxhip;

namespace {

// The context's device is current while a call lasts, the caller's again behind it.
struct OnDevice {
    int was = -1;
    bool ok = false;
    explicit OnDevice(int device) { ok = hipGetDevice(&was) == hipSuccess && (was == device || hipSetDevice(device) == hipSuccess); }
    ~OnDevice() {
        int now = -1;
        if (ok && hipGetDevice(&now) == hipSuccess && now != was) (void)hipSetDevice(was);
    }
};

bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// What is wrong with a cache and a batch, or nullptr.
const char* check(const oxhip_kv_cache* kv, const oxhip_kv_batch* b, KvView* kvv, KvBatchView* bv) {
    if (!kv || !b || !kv->k || !kv->v || !kv->k_scale || !kv->v_scale || !b->kv_len || !b->pages) return "null argument";
    if (!aligned(kv->k, 16) || !aligned(kv->v, 16)) return "k and v begin at multiples of 16 bytes";
    if (!aligned(kv->k_scale, 4) || !aligned(kv->v_scale, 4) || !aligned(b->kv_len, 4) || !aligned(b->pages, 4) || !aligned(b->row_start, 4)) return "an array of 4-byte values at an odd address";
    if (!kv->d || kv->d % 32 || kv->d > KV_MAX_D) return "d is a multiple of 32, 256 at most";
    const size_t page = kv->page_tokens;
    if (page < KV_BLOCK || page > ((size_t)1 << 30) || (page & (page - 1))) return "a page holds a power of two of tokens, 32 at least and 2^30 at most";
    if (!kv->n_kv || kv->n_kv > 16384 || !kv->n_pages || kv->n_pages > 0x7FFFFFFFu) return "1 to 16384 key heads, 1 to 2^31 - 1 pages";
    if (!b->n_seqs || !b->max_pages || b->max_pages > 0x7FFFFFFFu || b->max_pages > ((size_t)0x7FFFFFC0u) / page) return "sequences and pages: at least one, and fewer than 2^31 - 64 tokens in a sequence's table";
    if (b->n_seqs > ((size_t)1 << 24) || b->rows > ((size_t)1 << 28)) return "2^24 sequences and 2^28 rows at most";
    if (!b->row_start && b->rows != b->n_seqs) return "without row_start, every sequence has one row";
    uint32_t shift = 0;
    while (((size_t)KV_BLOCK << shift) < page) shift++;
    if (kv->n_pages > (((size_t)0x7FFFFFFFu / kv->n_kv) >> shift)) return "a cache has fewer than 2^31 blocks";
    *kvv = KvView{kv->k, kv->v, kv->k_scale, kv->v_scale, (uint32_t)kv->n_pages, (uint32_t)kv->n_kv, (uint32_t)kv->d, shift};
    *bv = KvBatchView{b->row_start, b->kv_len, b->pages, (uint32_t)b->n_seqs, (uint32_t)b->rows, (uint32_t)b->max_pages};
    return nullptr;
}

bool refuse(const char* who, const char* why) {
    set_error(std::string(who) + ": " + why);
    return false;
}

// The decode scratch of the calling stream, for the parts of results that workgroups leave for each other.
DecodeScratch* parts(oxhip_ctx* c, hipStream_t s, const char* who) {
    StreamScratch* sc = scratch_for(c, s, true);
    if (sc) return &sc->dec;
    set_error(std::string(who) + (stream_recording(s) ? ": the stream's scratch does not exist yet and a plan records on it (run the chain once before recording)" : ": device memory short"));
    return nullptr;
}

// What the calls of the attention have alike: the checks, and what the kernels get. nullptr, or what is wrong.
const char* check_attend(const oxhip_kv_cache* kv, const oxhip_kv_batch* b, const void* q, size_t q_stride, size_t n_q, int dtype, float scale, const oxhip_attend_rules* rules,
                         void* out, size_t out_stride, KvView* kvv, KvBatchView* bv, AttendCall* call) {
    if (!q || !out) return "null argument";
    if (const char* why = check(kv, b, kvv, bv)) return why;
    if (dtype != OXHIP_F32 && dtype != OXHIP_BF16) return "rows are f32 or bf16";
    if (!n_q || n_q % kv->n_kv || n_q > 65536) return "the query heads are a multiple of the key heads, 65536 at most";
    if (!(std::fabs(scale) <= 0x1p120f)) return "the scale lies within -2^120 and 2^120";
    const size_t size = dtype == OXHIP_BF16 ? 2 : 4, width = n_q * kv->d;
    if (!aligned(q, size) || !aligned(out, size)) return "rows begin at multiples of their values' size";
    if ((q_stride && q_stride < width) || (out_stride && out_stride < width)) return "rows lie at least a row apart";
    if (q == out) return "out lies apart from q";
    if (rules) {
        if (!(rules->cap == 0.0f || (rules->cap >= 0x1p-60f && rules->cap <= 0x1p60f))) return "a cap lies within 2^-60 and 2^60, or is 0 for none";
        if (!aligned(rules->slopes, 4) || !aligned(rules->prefix, 4) || !aligned(rules->first, 4)) return "an array of 4-byte values at an odd address";
        call->cap = rules->cap;
        call->slopes = rules->slopes;
        call->window = rules->window < 0x7FFFFFFFu ? (uint32_t)rules->window : 0;  // (no sequence is that long)
        call->prefix = rules->prefix;
        call->first = rules->first;
    }
    call->q = q;
    call->out = out;
    call->q_stride = q_stride ? q_stride : width;
    call->out_stride = out_stride ? out_stride : width;
    call->scale = scale;
    call->n_q = (uint32_t)n_q;
    call->bf16 = dtype == OXHIP_BF16;
    return nullptr;
}
// The groups of a batch whose sequences share first tokens: nullptr, or what is wrong.
const char* check_shared(const oxhip_kv_shared* shared, SharedView* v) {
    if (!shared || !shared->group_start || !shared->common) return "null argument";
    if (!aligned(shared->group_start, 4) || !aligned(shared->common, 4)) return "an array of 4-byte values at an odd address";
    if (!shared->n_groups || shared->n_groups > ((size_t)1 << 24)) return "1 to 2^24 groups";
    *v = SharedView{shared->group_start, shared->common, (uint32_t)shared->n_groups};
    return nullptr;
}
// A summary of a cache, or nullptr and what is wrong.
const char* check_summary(const oxhip_kv_cache* kv, const oxhip_kv_summary* sum, uint32_t* span_shift) {
    if (!sum || !sum->code || !sum->scale) return "null argument";
    if (!aligned(sum->code, 16) || !aligned(sum->scale, 4)) return "code begins at a multiple of 16 bytes, scale of 4";
    if (sum->span < KV_BLOCK || (sum->span & (sum->span - 1)) || sum->span > kv->page_tokens) return "a span is a power of two of tokens, 32 at least and a page at most";
    *span_shift = 0;
    while (((size_t)KV_BLOCK << *span_shift) < sum->span) ++*span_shift;
    return nullptr;
}

int append(const char* who, oxhip_ctx* c, const oxhip_kv_cache* kv, const oxhip_kv_batch* b, const SharedView& shared, const void* k, size_t k_stride, const void* v, size_t v_stride,
           const void* q, size_t q_stride, void* q_out, size_t q_out_stride, size_t n_q, int dtype, const oxhip_rope* rope, void* stream) {
    KvView kvv;
    KvBatchView bv;
    if (!k || !v) return refuse(who, "null argument");
    if (const char* why = check(kv, b, &kvv, &bv)) return refuse(who, why);
    if (dtype != OXHIP_F32 && dtype != OXHIP_BF16) return refuse(who, "rows are f32 or bf16");
    if ((n_q != 0) != (q != nullptr) || (n_q != 0) != (q_out != nullptr)) return refuse(who, "q, q_out and n_q: all of them, or none");
    if (n_q > 32768) return refuse(who, "32768 query heads at most");
    const size_t size = dtype == OXHIP_BF16 ? 2 : 4, width = kv->n_kv * kv->d, q_width = n_q * kv->d;
    if (!aligned(k, size) || !aligned(v, size) || !aligned(q, size) || !aligned(q_out, size)) return refuse(who, "rows begin at multiples of their values' size");
    if ((k_stride && k_stride < width) || (v_stride && v_stride < width) || (q_stride && q_stride < q_width) || (q_out_stride && q_out_stride < q_width))
        return refuse(who, "rows lie at least a row apart");
    if (q && q == q_out && (q_stride ? q_stride : q_width) != (q_out_stride ? q_out_stride : q_width)) return refuse(who, "in place, q and q_out have one stride");
    RopeView r{};
    if (rope) {
        if (!rope->table || !aligned(rope->table, 8) || !rope->n_pos || rope->n_pos > 0x7FFFFFFFu || !rope->n_rot || rope->n_rot % 2 || rope->n_rot > kv->d)
            return refuse(who, "a table of angles at a multiple of 8 bytes, an even number of rotated channels, at most d");
        r = RopeView{rope->table, (uint32_t)rope->n_pos, (uint32_t)(rope->n_rot / 2), rope->interleaved ? 1u : 0u};
    }
    const size_t heads = 2 * kv->n_kv + n_q;
    if (!kv_launch_fits(kv_append_workgroups(b->row_start, b->rows, b->n_seqs, heads), 256, b->row_start ? heads : 1))
        return refuse(who, "more rows, sequences or heads than one launch takes (2^24 workgroups; with row_start 65535 heads)");
    if (!c) return refuse(who, "null context");
    if (!b->rows) return 1;
    OnDevice on(c->device);
    if (!on.ok) return refuse(who, "hipSetDevice failed");
    HIP_TRY(launch_kv_append(kvv, bv, shared, r, k, k_stride ? k_stride : width, v, v_stride ? v_stride : width, q, q_stride ? q_stride : q_width, q_out, q_out_stride ? q_out_stride : q_width,
                             (uint32_t)n_q, dtype == OXHIP_BF16, static_cast<hipStream_t>(stream)),
            "kv_append launch");
    return 1;
}

}  // namespace

extern "C" {

int oxhip_dev_kv_append(oxhip_ctx* c, const oxhip_kv_cache* kv, const oxhip_kv_batch* b, const void* k, size_t k_stride, const void* v, size_t v_stride, const void* q,
                        size_t q_stride, void* q_out, size_t q_out_stride, size_t n_q, int dtype, const oxhip_rope* rope, void* stream) {
    return append("kv_append", c, kv, b, SharedView{}, k, k_stride, v, v_stride, q, q_stride, q_out, q_out_stride, n_q, dtype, rope, stream);
}

int oxhip_dev_kv_append_shared(oxhip_ctx* c, const oxhip_kv_cache* kv, const oxhip_kv_batch* b, const oxhip_kv_shared* shared, const void* k, size_t k_stride, const void* v,
                               size_t v_stride, const void* q, size_t q_stride, void* q_out, size_t q_out_stride, size_t n_q, int dtype, const oxhip_rope* rope, void* stream) {
    const char* who = "kv_append_shared";
    SharedView sv{};
    if (const char* why = check_shared(shared, &sv)) return refuse(who, why);
    return append(who, c, kv, b, sv, k, k_stride, v, v_stride, q, q_stride, q_out, q_out_stride, n_q, dtype, rope, stream);
}

int oxhip_dev_kv_read(oxhip_ctx* c, const oxhip_kv_cache* kv, const oxhip_kv_batch* b, size_t count, void* k_out, void* v_out, int dtype, void* stream) {
    const char* who = "kv_read";
    KvView kvv;
    KvBatchView bv;
    if (!k_out && !v_out) return refuse(who, "null argument");
    if (const char* why = check(kv, b, &kvv, &bv)) return refuse(who, why);
    if (dtype != OXHIP_F32 && dtype != OXHIP_BF16) return refuse(who, "values are f32 or bf16");
    const size_t size = dtype == OXHIP_BF16 ? 2 : 4;
    if (!aligned(k_out, size) || !aligned(v_out, size)) return refuse(who, "values begin at multiples of their size");
    if (count > 0x7FFFFFC0u || !kv_launch_fits(kv_read_blocks(count) * b->n_seqs, 256)) return refuse(who, "more tokens than one launch takes (2^24 blocks)");
    if (!c) return refuse(who, "null context");
    if (!count) return 1;
    OnDevice on(c->device);
    if (!on.ok) return refuse(who, "hipSetDevice failed");
    HIP_TRY(launch_kv_read(kvv, bv, count, k_out, v_out, dtype == OXHIP_BF16, static_cast<hipStream_t>(stream)), "kv_read launch");
    return 1;
}

int oxhip_dev_attend(oxhip_ctx* c, const oxhip_kv_cache* kv, const oxhip_kv_batch* b, const void* q, size_t q_stride, size_t n_q, int dtype, float scale,
                     const oxhip_attend_rules* rules, void* out, size_t out_stride, void* stream) {
    const char* who = "attend";
    KvView kvv;
    KvBatchView bv;
    AttendCall call{};
    if (const char* why = check_attend(kv, b, q, q_stride, n_q, dtype, scale, rules, out, out_stride, &kvv, &bv, &call)) return refuse(who, why);
    const size_t g = n_q / kv->n_kv;
    if (b->row_start && b->n_seqs == 1 ? !kv_launch_fits(kv_places(b->rows * g, 1, 128, 1) * kv->n_kv, 256)
                                       : !kv_launch_fits(kv_units(b->row_start, b->rows, b->n_seqs, g, kv->n_kv), 512))
        return refuse(who, "more rows, sequences or heads than one launch takes");
    if (!c) return refuse(who, "null context");
    if (!b->rows) return 1;
    OnDevice on(c->device);
    if (!on.ok) return refuse(who, "hipSetDevice failed");
    hipStream_t s = static_cast<hipStream_t>(stream);
    DecodeScratch* sc = parts(c, s, who);
    if (!sc) return 0;
    HIP_TRY(launch_attend(kvv, bv, call, *sc, s), "attend launch");
    return 1;
}

int oxhip_dev_attend_shared(oxhip_ctx* c, const oxhip_kv_cache* kv, const oxhip_kv_batch* b, const oxhip_kv_shared* shared, const void* q, size_t q_stride, size_t n_q, int dtype,
                            float scale, const oxhip_attend_rules* rules, void* out, size_t out_stride, void* stream) {
    const char* who = "attend_shared";
    KvView kvv;
    KvBatchView bv;
    AttendCall call{};
    if (const char* why = check_attend(kv, b, q, q_stride, n_q, dtype, scale, rules, out, out_stride, &kvv, &bv, &call)) return refuse(who, why);
    SharedView sv{};
    if (const char* why = check_shared(shared, &sv)) return refuse(who, why);
    if (!kv_launch_fits(kv_row_tiles(b->rows, n_q / kv->n_kv, true) * kv->n_kv, 512)) return refuse(who, "more rows or heads than one launch takes");
    if (!c) return refuse(who, "null context");
    if (!b->rows) return 1;
    OnDevice on(c->device);
    if (!on.ok) return refuse(who, "hipSetDevice failed");
    hipStream_t s = static_cast<hipStream_t>(stream);
    DecodeScratch* sc = parts(c, s, who);
    if (!sc) return 0;
    HIP_TRY(launch_attend_shared(kvv, bv, sv, call, *sc, s), "attend_shared launch");
    return 1;
}

int oxhip_dev_kv_summarize(oxhip_ctx* c, const oxhip_kv_cache* kv, const oxhip_kv_batch* b, const oxhip_kv_summary* sum, void* stream) {
    const char* who = "kv_summarize";
    SummaryArgs a{};
    if (const char* why = check(kv, b, &a.kv, &a.b)) return refuse(who, why);
    if (const char* why = check_summary(kv, sum, &a.span_shift)) return refuse(who, why);
    if (!kv_launch_fits((b->row_start ? kv_places(b->rows, b->n_seqs, (uint32_t)sum->span, 2) : b->n_seqs) * kv->n_kv, 256)) return refuse(who, "more rows, sequences or heads than one launch takes");
    if (!c) return refuse(who, "null context");
    if (!b->rows) return 1;
    a.code = sum->code;
    a.scale = sum->scale;
    OnDevice on(c->device);
    if (!on.ok) return refuse(who, "hipSetDevice failed");
    HIP_TRY(launch_kv_summarize(a, static_cast<hipStream_t>(stream)), "kv_summarize launch");
    return 1;
}

int oxhip_dev_kv_summary_read(oxhip_ctx* c, const oxhip_kv_cache* kv, const oxhip_kv_batch* b, const oxhip_kv_summary* sum, size_t count, float* out, void* stream) {
    const char* who = "kv_summary_read";
    SummaryArgs a{};
    if (!out) return refuse(who, "null argument");
    if (const char* why = check(kv, b, &a.kv, &a.b)) return refuse(who, why);
    if (const char* why = check_summary(kv, sum, &a.span_shift)) return refuse(who, why);
    if (!aligned(out, 16)) return refuse(who, "out begins at a multiple of 16 bytes");
    if (count > 0x7FFFFFFFu || (count && b->n_seqs * kv->n_kv > 0xFFFFFFFFu / (kv->d / 4) / count)) return refuse(who, "more spans than one launch takes");
    if (!c) return refuse(who, "null context");
    if (!count) return 1;
    a.code = sum->code;
    a.scale = sum->scale;
    OnDevice on(c->device);
    if (!on.ok) return refuse(who, "hipSetDevice failed");
    HIP_TRY(launch_kv_summary_read(a, count, out, static_cast<hipStream_t>(stream)), "kv_summary_read launch");
    return 1;
}

int oxhip_dev_kv_select(oxhip_ctx* c, const oxhip_kv_cache* kv, const oxhip_kv_batch* b, const oxhip_kv_summary* sum, const void* q, size_t q_stride, size_t n_q, int dtype,
                        size_t count, size_t first, size_t last, int32_t* chosen, void* stream) {
    const char* who = "kv_select";
    SelectArgs a{};
    if (!q || !chosen) return refuse(who, "null argument");
    if (const char* why = check(kv, b, &a.kv, &a.b)) return refuse(who, why);
    if (const char* why = check_summary(kv, sum, &a.span_shift)) return refuse(who, why);
    if (dtype != OXHIP_F32 && dtype != OXHIP_BF16) return refuse(who, "rows are f32 or bf16");
    if (!n_q || n_q % kv->n_kv || n_q > 65536) return refuse(who, "the query heads are a multiple of the key heads, 65536 at most");
    const size_t width = n_q * kv->d;
    if (!aligned(q, dtype == OXHIP_BF16 ? 2 : 4) || !aligned(chosen, 4)) return refuse(who, "rows begin at multiples of their values' size");
    if (q_stride && q_stride < width) return refuse(who, "rows lie at least a row apart");
    if (!count || count > SELECT_SPANS || first > count || last > count - first) return refuse(who, "1 to 16384 spans of a row, the first and the last ones among them");
    if (b->max_pages > SELECT_SPANS / (kv->page_tokens / sum->span)) return refuse(who, "a sequence's table has room for 16384 spans at most");
    if (!kv_launch_fits((b->row_start ? kv_places(b->rows, b->n_seqs, 1, 1) : b->n_seqs) * kv->n_kv, 1024)) return refuse(who, "more rows, sequences or heads than one launch takes");
    if (!c) return refuse(who, "null context");
    if (!b->rows) return 1;
    a.code = sum->code;
    a.scale = sum->scale;
    a.q = q;
    a.q_stride = q_stride ? q_stride : width;
    a.out = chosen;
    a.g = (uint32_t)(n_q / kv->n_kv);
    a.count = (uint32_t)count;
    a.first = (uint32_t)first;
    a.last = (uint32_t)last;
    OnDevice on(c->device);
    if (!on.ok) return refuse(who, "hipSetDevice failed");
    HIP_TRY(launch_kv_select(a, dtype == OXHIP_BF16, static_cast<hipStream_t>(stream)), "kv_select launch");
    return 1;
}

int oxhip_dev_attend_selected(oxhip_ctx* c, const oxhip_kv_cache* kv, const oxhip_kv_batch* b, const int32_t* chosen, size_t count, size_t span, const void* q, size_t q_stride,
                              size_t n_q, int dtype, float scale, const oxhip_attend_rules* rules, void* out, size_t out_stride, void* stream) {
    const char* who = "attend_selected";
    KvView kvv;
    KvBatchView bv;
    AttendCall call{};
    if (const char* why = check_attend(kv, b, q, q_stride, n_q, dtype, scale, rules, out, out_stride, &kvv, &bv, &call)) return refuse(who, why);
    if (!chosen) return refuse(who, "null argument");
    if (!aligned(chosen, 4)) return refuse(who, "an array of 4-byte values at an odd address");
    if (span < KV_BLOCK || (span & (span - 1)) || span > kv->page_tokens) return refuse(who, "a span is a power of two of tokens, 32 at least and a page at most");
    if (!count || count > ((size_t)1 << 26) / (span / KV_BLOCK)) return refuse(who, "1 span of a row at least, 2^31 tokens of them at most");
    if (!kv_launch_fits(kv_row_tiles(b->rows, n_q / kv->n_kv, false) * kv->n_kv, 512)) return refuse(who, "more rows or heads than one launch takes");
    if (!c) return refuse(who, "null context");
    if (!b->rows) return 1;
    OnDevice on(c->device);
    if (!on.ok) return refuse(who, "hipSetDevice failed");
    hipStream_t s = static_cast<hipStream_t>(stream);
    DecodeScratch* sc = parts(c, s, who);
    if (!sc) return 0;
    HIP_TRY(launch_attend_selected(kvv, bv, ChosenView{chosen, (uint32_t)count, (uint32_t)(span / KV_BLOCK)}, call, *sc, s), "attend_selected launch");
    return 1;
}

int oxhip_dev_sample(oxhip_ctx* c, const void* logits, size_t stride, size_t rows, size_t vocab, int dtype, const oxhip_sample_rules* rules, const float* u, int32_t* next,
                     float* logp, void* stream) {
    const char* who = "sample";
    if (!logits || !u || !next) return refuse(who, "null argument");
    if (dtype != OXHIP_F32 && dtype != OXHIP_BF16) return refuse(who, "logits are f32 or bf16");
    if (!vocab || vocab > 0x7FFFF000u || rows > ((size_t)1 << 22) - 1) return refuse(who, "a vocabulary of 1 to 2^31 - 4096, fewer than 2^22 rows");
    if (!aligned(logits, dtype == OXHIP_BF16 ? 2 : 4) || !aligned(u, 4) || !aligned(next, 4) || !aligned(logp, 4)) return refuse(who, "rows begin at multiples of their values' size");
    if (stride && stride < vocab) return refuse(who, "rows lie at least a row apart");
    SampleArgs a{};
    a.x = logits;
    a.stride = stride ? stride : vocab;
    a.rows = (uint32_t)rows;
    a.vocab = (uint32_t)vocab;
    a.u = u;
    a.next = next;
    a.logp = logp;
    if (rules) {
        for (const void* p : {(const void*)rules->temperature, (const void*)rules->top_k, (const void*)rules->top_p, (const void*)rules->min_p})
            if (!aligned(p, 4)) return refuse(who, "an array of 4-byte values at an odd address");
        a.temperature = rules->temperature;
        a.top_k = rules->top_k;
        a.top_p = rules->top_p;
        a.min_p = rules->min_p;
    }
    if (!c) return refuse(who, "null context");
    if (!rows) return 1;
    OnDevice on(c->device);
    if (!on.ok) return refuse(who, "hipSetDevice failed");
    hipStream_t s = static_cast<hipStream_t>(stream);
    DecodeScratch* sc = parts(c, s, who);
    if (!sc) return 0;
    HIP_TRY(launch_sample(a, dtype == OXHIP_BF16, *sc, s), "sample launch");
    return 1;
}

int oxhip_dev_logits(oxhip_ctx* c, const void* logits, size_t stride, void* out, size_t out_stride, size_t rows, size_t vocab, int dtype, const oxhip_logit_rules* rules,
                     int32_t* next, void* stream) {
    const char* who = "logits";
    if (!logits || (!out && !next)) return refuse(who, "null argument");
    if (dtype != OXHIP_F32 && dtype != OXHIP_BF16) return refuse(who, "logits are f32 or bf16");
    const size_t size = dtype == OXHIP_BF16 ? 2 : 4;
    if (!vocab || vocab > 0x7FFFF000u || rows > ((size_t)1 << 24)) return refuse(who, "a vocabulary of 1 to 2^31 - 4096, 2^24 rows at most");
    if (!aligned(logits, size) || !aligned(out, size) || !aligned(next, 4)) return refuse(who, "rows begin at multiples of their values' size");
    if ((stride && stride < vocab) || (out_stride && out_stride < vocab)) return refuse(who, "rows lie at least a row apart");
    LogitArgs a{};
    a.x = logits;
    a.out = out;
    a.next = next;
    a.x_stride = stride ? stride : vocab;
    a.out_stride = out_stride ? out_stride : vocab;
    if (out == logits && a.x_stride != a.out_stride) return refuse(who, "in place, there is one stride");
    a.rows = (uint32_t)rows;
    a.vocab = (uint32_t)vocab;
    if (rules) {
        const oxhip_logit_rules& r = *rules;
        if ((r.history != nullptr) != (r.history_len != nullptr) || (r.history && !r.history_stride)) return refuse(who, "a history has a length for each row, and room for a token");
        if (!r.history && (r.prompt_len || r.repetition || r.presence || r.frequency)) return refuse(who, "penalties need a history");
        if ((r.bias_start != nullptr) != (r.bias_id != nullptr) || (r.bias_start != nullptr) != (r.bias != nullptr)) return refuse(who, "bias_start, bias_id and bias: all of them, or none");
        if (r.n_bias > 0x7FFFFFFFu) return refuse(who, "2^31 - 1 biases at most");
        if (r.allowed ? r.allowed_stride < (vocab + 31) / 32 || !r.n_allowed || r.n_allowed > 0x7FFFFFFFu : r.allowed_row != nullptr) return refuse(who, "masks of (vocab + 31) / 32 words at least, and as many as there are");
        if (r.allowed && !r.allowed_row && r.n_allowed < rows) return refuse(who, "a mask for each row, or allowed_row");
        for (const void* p : {(const void*)r.history, (const void*)r.history_len, (const void*)r.prompt_len, (const void*)r.repetition, (const void*)r.presence, (const void*)r.frequency,
                              (const void*)r.bias_start, (const void*)r.bias_id, (const void*)r.bias, (const void*)r.allowed, (const void*)r.allowed_row})
            if (!aligned(p, 4)) return refuse(who, "an array of 4-byte values at an odd address");
        if (r.repetition || r.presence || r.frequency) {
            a.history = r.history;
            a.history_len = r.history_len;
            a.prompt_len = r.prompt_len;
            a.history_stride = r.history_stride;
            a.repetition = r.repetition;
            a.presence = r.presence;
            a.frequency = r.frequency;
        }
        a.bias_start = r.bias_start;
        a.bias_id = r.bias_id;
        a.bias = r.bias;
        a.n_bias = (uint32_t)r.n_bias;
        a.allowed = r.allowed;
        a.allowed_stride = r.allowed_stride;
        a.n_allowed = (uint32_t)r.n_allowed;
        a.allowed_row = r.allowed_row;
    }
    if (!kv_launch_fits(rows * logit_slices(vocab), LOGIT_THREADS)) return refuse(who, "more logits than one launch takes (2^23 slices of 4096)");
    const char* too_many = "with next, 16384 rows at most, and 2^21 slices of 4096 logits in all of them";
    if (next && (rows > LOGIT_NEXT_ROWS || rows * logit_slices(vocab) > LOGIT_NEXT_SLICES)) return refuse(who, too_many);
    if (!c) return refuse(who, "null context");
    if (!rows) return 1;
    OnDevice on(c->device);
    if (!on.ok) return refuse(who, "hipSetDevice failed");
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (next) {
        DecodeScratch* sc = parts(c, s, who);
        if (!sc) return 0;
        if (rows * CTR_STRIDE > sc->ncounters || rows * logit_slices(vocab) * 2 > sc->partial_floats) return refuse(who, too_many);
        a.best = reinterpret_cast<uint64_t*>(sc->partial);
        a.counters = sc->counters;
    }
    HIP_TRY(launch_logits(a, dtype == OXHIP_BF16, s), "logits launch");
    return 1;
}

}  // extern "C"

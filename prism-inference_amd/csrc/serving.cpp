// serving.cpp -- the paged 8-bit cache of the C ABI: argument checks, scratch and launches of
// kvcache.hip and paged_attention.hip.
#include <cmath>
#include <new>

#include "runtime_internal.hpp"
#include "serving.hpp"

using namespace prism;
using namespace prism::rt;

struct prism_hip_rope {
    prism_hip_ctx *ctx = nullptr;
    Rotation rot;
    double *freq = nullptr;
};

namespace {

// Device allocations and launches go to the context's device, whichever is current.
struct OnDevice {
    int before = -1;
    explicit OnDevice(const prism_hip_ctx *c) {
        int now = -1;
        if (c && hipGetDevice(&now) == hipSuccess && now != c->device && hipSetDevice(c->device) == hipSuccess) before = now;
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;
};

// Bounds that keep every grid below 2^32 work-items.
constexpr uint64_t kMostTokens = 1u << 23, kMostHeads = 1u << 12, kMostRows = 1u << 26;

bool aligned(const void *p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
size_t type_size(int dtype) { return dtype == PRISM_DTYPE_F32 ? 4 : 2; }
bool head_dim_ok(uint32_t d) { return d == 64 || d == 128 || d == 256; }
bool page_ok(uint32_t p) { return p >= 16 && p <= 256 && (p & (p - 1)) == 0; }

int bad(prism_hip_ctx *c, const char *what) { return fail(c, PRISM_ERR_INVALID_INPUT, what); }

// What every entry point asks first.
int enter(prism_hip_ctx *c, void *stream, hipStream_t *s) {
    const int rc = check_ready(c);
    return rc ? rc : call_stream(c, stream, s);
}

int check_cache(prism_hip_ctx *c, const prism_kv_cache *k) {
    if (!k || !k->k || !k->v || !k->k_scale || !k->v_scale) return bad(c, "null cache");
    if (k->format != PRISM_CACHE_INT8 && k->format != PRISM_CACHE_E4M3) return bad(c, "unknown cache format");
    if (!head_dim_ok(k->head_dim)) return fail(c, PRISM_ERR_UNSUPPORTED, "cache head_dim must be 64, 128 or 256");
    if (!page_ok(k->page_size)) return fail(c, PRISM_ERR_UNSUPPORTED, "cache page_size must be 16, 32, 64, 128 or 256");
    if (!k->pages || static_cast<uint64_t>(k->pages) * k->page_size > 0x7fffffffull) return bad(c, "cache needs 1 .. 2^31 - 1 positions");
    if (!k->kv_heads || k->kv_heads > kMostHeads) return bad(c, "cache kv_heads out of range");
    if (!aligned(k->k, 16) || !aligned(k->v, 16) || !aligned(k->k_scale, 4) || !aligned(k->v_scale, 4))
        return bad(c, "cache codes must be 16-byte aligned");
    return PRISM_OK;
}

// Rows [tokens][heads][head_dim]: not null, aligned to their type, and not overlapping.
int check_rows(prism_hip_ctx *c, int dtype, const void *p, uint64_t stride, uint64_t heads, uint32_t head_dim) {
    if (!p) return bad(c, "null device pointer");
    if (!aligned(p, type_size(dtype))) return bad(c, "rows not aligned to their type");
    if (stride < heads * head_dim || stride > (1ull << 40)) return bad(c, "row stride below heads * head_dim");
    return PRISM_OK;
}

int check_dtype(prism_hip_ctx *c, int dtype) {
    return dtype == PRISM_DTYPE_F32 || dtype == PRISM_DTYPE_F16 || dtype == PRISM_DTYPE_BF16 ? PRISM_OK : bad(c, "unknown element type");
}
int check_eps(prism_hip_ctx *c, float eps) { return std::isfinite(eps) && eps >= 0.0f ? PRISM_OK : bad(c, "eps must be finite and not negative"); }
int check_counts(prism_hip_ctx *c, uint64_t tokens, uint64_t heads) {
    return tokens <= kMostTokens && heads && heads <= kMostHeads && tokens * heads <= kMostRows ? PRISM_OK : bad(c, "tokens or heads out of range");
}

int check_rope(prism_hip_ctx *c, const prism_hip_rope *rope, uint32_t head_dim) {
    if (!rope || rope->ctx != c) return bad(c, "rotation missing, or another context's");
    return rope->rot.dims <= head_dim ? PRISM_OK : bad(c, "rotation wider than the head");
}

}  // namespace

extern "C" {

int prism_hip_kv_plan_device(prism_hip_ctx *c, const prism_kv_plan *p, void *stream) {
    CaptureNote note(c);
    hipStream_t s;
    int rc = enter(c, stream, &s);
    if (rc) return rc;
    if (!p || !p->lengths || !p->added || !p->block_table || !p->free_pages || !p->free_count || !p->new_lengths || !p->offsets ||
        !p->positions || !p->slots || !p->owners || !p->counts)
        return bad(c, "null device pointer");
    if (!p->requests || p->requests > kMostTokens || !p->max_tokens || p->max_tokens > kMostTokens || !p->max_pages ||
        p->free_capacity > 0x7fffffffu)
        return bad(c, "requests, tokens or pages out of range");
    if (!page_ok(p->page_size)) return fail(c, PRISM_ERR_UNSUPPORTED, "page_size must be 16, 32, 64, 128 or 256");
    if (static_cast<uint64_t>(p->max_pages) * p->page_size > 0x7fffffffull) return bad(c, "max_pages * page_size out of range");
    OnDevice on(c);
    rc = ensure(c, c->plan, plan_scratch_bytes(p->requests));
    return rc ? rc : launch_result(c, launch_kv_plan(*p, c->plan.p, c->err, s), "plan launch");
}

int prism_hip_rope_frequencies(uint32_t dims, double base, double factor, double original, double alpha, double beta, double *out) {
    if (!out || dims < 2 || dims > 256 || dims % 2 || !(base > 0.0) || !std::isfinite(base) || !(factor >= 1.0) || !std::isfinite(factor))
        return PRISM_ERR_INVALID_INPUT;
    const bool banded = original != 0.0;
    if (banded && (!(original > 0.0) || !std::isfinite(original) || !(alpha < beta) || !std::isfinite(alpha) || !std::isfinite(beta)))
        return PRISM_ERR_INVALID_INPUT;
    for (uint32_t i = 0; i < dims / 2; ++i) {
        const double f = std::pow(base, -2.0 * i / dims);
        double keep = 0.0;
        if (banded) {
            const double turns = original * f / (2.0 * 3.14159265358979323846);
            keep = std::fmin(std::fmax((turns - alpha) / (beta - alpha), 0.0), 1.0);
        }
        out[i] = (1.0 - keep) * f / factor + keep * f;
    }
    return PRISM_OK;
}

prism_hip_rope *prism_hip_rope_create(prism_hip_ctx *c, uint32_t dims, int interleaved, const double *frequencies, double magnitude) {
    if (check_live(c)) return nullptr;
    bool ok = frequencies && dims >= 2 && dims <= 256 && dims % 2 == 0 && std::isfinite(magnitude);
    for (uint32_t i = 0; ok && i < dims / 2; ++i) ok = std::isfinite(frequencies[i]) && std::fabs(frequencies[i]) <= 1e6;
    if (!ok) {
        fail(c, PRISM_ERR_INVALID_INPUT, "unsupported rotation");
        return nullptr;
    }
    OnDevice on(c);
    auto *r = new (std::nothrow) prism_hip_rope;
    if (!r) {
        fail(c, PRISM_ERR_RESOURCE, "out of memory");
        return nullptr;
    }
    const size_t bytes = sizeof(double) * (dims / 2);
    hipError_t e = hipMalloc(&r->freq, bytes);
    if (e == hipSuccess) {
        e = hipMemcpy(r->freq, frequencies, bytes, hipMemcpyHostToDevice);
        if (e != hipSuccess) (void)hipFree(r->freq);
    }
    if (e != hipSuccess) {
        hip_fail(c, e, "rotation table");
        delete r;
        return nullptr;
    }
    r->ctx = c;
    r->rot = Rotation{r->freq, dims, interleaved != 0, magnitude};
    return r;
}

void prism_hip_rope_destroy(prism_hip_rope *r) {
    if (!r) return;
    OnDevice on(r->ctx);
    (void)hipStreamSynchronize(r->ctx->stream);
    (void)hipFree(r->freq);
    delete r;
}

int prism_hip_rope_device(prism_hip_ctx *c, const prism_hip_rope *rope, int dtype, const void *x, uint64_t x_stride,
                          const int32_t *positions, uint32_t tokens, uint32_t heads, uint32_t head_dim, const float *norm, float eps,
                          void *out, uint64_t out_stride, void *stream) {
    hipStream_t s;
    int rc = enter(c, stream, &s);
    if (!rc && !head_dim_ok(head_dim)) rc = fail(c, PRISM_ERR_UNSUPPORTED, "head_dim must be 64, 128 or 256");
    if (!rc) rc = check_dtype(c, dtype);
    if (!rc) rc = check_counts(c, tokens, heads);
    if (!rc) rc = check_eps(c, eps);
    if (!rc) rc = check_rope(c, rope, head_dim);
    if (rc || tokens == 0) return rc;
    rc = check_rows(c, dtype, x, x_stride, heads, head_dim);
    if (!rc) rc = check_rows(c, dtype, out, out_stride, heads, head_dim);
    if (!rc && !positions) rc = bad(c, "null device pointer");
    if (!rc && x == out && x_stride != out_stride) rc = bad(c, "rotation in place needs one stride");
    if (rc) return rc;
    OnDevice on(c);
    const RopeRows a{x, out, x_stride, out_stride, heads, norm};
    return launch_result(c, launch_rope(dtype, rope->rot, a, RopeRows{}, positions, tokens, head_dim, eps, c->err, s), "rotation launch");
}

static int check_append(prism_hip_ctx *c, const prism_kv_cache *cache, int dtype, const void *k, uint64_t k_stride, const void *v,
                        uint64_t v_stride, const int32_t *slots, uint32_t tokens) {
    int rc = check_cache(c, cache);
    if (!rc) rc = check_dtype(c, dtype);
    if (!rc) rc = check_counts(c, tokens, cache->kv_heads);
    if (rc || tokens == 0) return rc;
    rc = check_rows(c, dtype, k, k_stride, cache->kv_heads, cache->head_dim);
    if (!rc) rc = check_rows(c, dtype, v, v_stride, cache->kv_heads, cache->head_dim);
    return rc || slots ? rc : bad(c, "null device pointer");
}

int prism_hip_kv_append_device(prism_hip_ctx *c, const prism_kv_cache *cache, int dtype, const void *k, uint64_t k_stride,
                               const void *v, uint64_t v_stride, const int32_t *slots, uint32_t tokens, void *stream) {
    hipStream_t s;
    int rc = enter(c, stream, &s);
    if (!rc) rc = check_append(c, cache, dtype, k, k_stride, v, v_stride, slots, tokens);
    if (rc || tokens == 0) return rc;
    OnDevice on(c);
    return launch_result(c, launch_kv_append(*cache, dtype, k, k_stride, v, v_stride, slots, tokens, c->err, s), "append launch");
}

int prism_hip_qkv_append_device(prism_hip_ctx *c, const prism_hip_rope *rope, const prism_kv_cache *cache, const prism_qkv_append *a,
                                void *stream) {
    CaptureNote note(c);
    hipStream_t s;
    int rc = enter(c, stream, &s);
    if (rc) return rc;
    if (!a) return bad(c, "null step");
    rc = check_append(c, cache, a->dtype, a->k, a->k_stride, a->v, a->v_stride, a->slots, a->tokens);
    if (!rc) rc = check_counts(c, a->tokens, a->heads);
    if (!rc) rc = check_eps(c, a->eps);
    if (!rc) rc = check_rope(c, rope, cache->head_dim);
    if (rc || a->tokens == 0) return rc;
    const uint32_t d = cache->head_dim, kv = cache->kv_heads;
    rc = check_rows(c, a->dtype, a->q, a->q_stride, a->heads, d);
    if (!rc) rc = check_rows(c, a->dtype, a->q_out, a->q_out_stride, a->heads, d);
    if (!rc && !a->positions) rc = bad(c, "null device pointer");
    if (!rc && a->q == a->q_out && a->q_stride != a->q_out_stride) rc = bad(c, "rotation in place needs one stride");
    if (rc) return rc;
    OnDevice on(c);
    const uint64_t width = static_cast<uint64_t>(kv) * d;
    rc = ensure(c, c->rope, type_size(a->dtype) * width * a->tokens);
    if (rc) return rc;
    const RopeRows q{a->q, a->q_out, a->q_stride, a->q_out_stride, a->heads, a->q_norm};
    const RopeRows k{a->k, c->rope.p, a->k_stride, width, kv, a->k_norm};
    rc = launch_result(c, launch_rope(a->dtype, rope->rot, q, k, a->positions, a->tokens, d, a->eps, c->err, s), "rotation launch");
    if (rc) return rc;
    return launch_result(c, launch_kv_append(*cache, a->dtype, c->rope.p, width, a->v, a->v_stride, a->slots, a->tokens, c->err, s),
                         "append launch");
}

int prism_hip_attention_device(prism_hip_ctx *c, const prism_kv_cache *cache, const prism_attention *a, void *stream) {
    CaptureNote note(c);
    hipStream_t s;
    int rc = enter(c, stream, &s);
    if (rc) return rc;
    if (!a) return bad(c, "null call");
    rc = check_cache(c, cache);
    if (!rc) rc = check_dtype(c, a->dtype);
    if (!rc) rc = check_counts(c, a->tokens, a->heads);
    if (rc) return rc;
    if (a->heads % cache->kv_heads) return bad(c, "heads must be a multiple of kv_heads");
    if (!std::isfinite(a->scale)) return bad(c, "scale must be finite");
    if (a->window && !a->causal) return bad(c, "a window needs the causal mask");
    if (a->window > 0x7fffffffu || a->max_length > 0x7fffffffu) return bad(c, "window or max_length out of range");
    if (static_cast<uint64_t>(a->requests) * cache->kv_heads > kMostTokens || !a->max_pages || static_cast<uint64_t>(a->max_pages) * cache->page_size > 0x7fffffffull)
        return bad(c, "requests or max_pages out of range");
    if (a->tokens == 0 || a->requests == 0) return PRISM_OK;
    rc = check_rows(c, a->dtype, a->q, a->q_stride, a->heads, cache->head_dim);
    if (!rc) rc = check_rows(c, a->dtype, a->out, a->out_stride, a->heads, cache->head_dim);
    if (rc) return rc;
    if (!a->offsets || !a->lengths || !a->block_table) return bad(c, "null device pointer");
    if (a->q == a->out && a->q_stride != a->out_stride) return bad(c, "attention in place needs one stride");
    OnDevice on(c);
    const size_t need = attention_scratch_bytes(*cache, *a, c->cus);
    if (need) rc = ensure(c, c->att, need);
    if (rc) return rc;
    return launch_result(c, launch_attention_paged(*cache, *a, c->att.p, c->cus, c->err, s), "attention launch");
}

}  // extern "C"

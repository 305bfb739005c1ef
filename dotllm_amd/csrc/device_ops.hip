// device_ops.hip -- the entry points of include/llmdot_hip_cache.h: operators
// over device memory, enqueued on the context's stream.
#include <math.h>
#include <string.h>

#include <new>
#include <string>

#include "../../include/llmdot_hip_cache.h"
#include "context.h"
#include "kernels.h"

using namespace llmdot;

struct llmdot_hip_kv_cache {
    llmdot_hip_ctx* ctx = nullptr;
    KvView view{};
};

namespace {

// The context's device for the call, the caller's afterwards.
struct OnDevice {
    int was = -1;
    hipError_t err;
    explicit OnDevice(int device) {
        err = hipGetDevice(&was);
        if (err == hipSuccess && was != device) err = hipSetDevice(device);
        else was = -1;
    }
    ~OnDevice() {
        if (was >= 0) (void)hipSetDevice(was);
    }
};

int device_error(const char* what, hipError_t e) {
    return ctx_fail(LLMDOT_E_DEVICE, std::string(what) + ": " + hipGetErrorString(e));
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The call's rows, checked; *total = batch * tokens.  A call of none is checked for
// its sizes only: empty arrays have no address.
int check_rows(const llmdot_hip_token_batch* rows, KvRows* out, int64_t* total) {
    if (!rows) return ctx_fail(LLMDOT_E_INVALID, "null token batch");
    if (rows->batch < 0 || rows->tokens < 0) return ctx_fail(LLMDOT_E_INVALID, "negative batch or tokens");
    if (rows->batch > MAX_SEQUENCES) return ctx_fail(LLMDOT_E_UNSUPPORTED, "more than 4096 sequences in a call");
    *total = (int64_t)rows->batch * rows->tokens;
    if (*total > 0 && (!rows->slots_dev || !rows->starts_dev)) return ctx_fail(LLMDOT_E_INVALID, "null slots or starts");
    *out = {rows->batch, rows->tokens, rows->slots_dev, rows->starts_dev, rows->counts_dev};
    return 0;
}

// A row stride in floats: 0 is packed.
int check_stride(const char* name, int64_t width, int64_t* stride) {
    if (*stride == 0) *stride = width;
    if (*stride < width || *stride % 4 != 0)
        return ctx_fail(LLMDOT_E_INVALID, std::string(name) + " stride must be 0 or a multiple of 4 of at least a row");
    return 0;
}

int check_array(const char* name, const void* p) {
    if (!p) return ctx_fail(LLMDOT_E_INVALID, std::string("null ") + name);
    if (!aligned(p)) return ctx_fail(LLMDOT_E_INVALID, std::string(name) + " is not 16-byte aligned");
    return 0;
}

// Workgroups of a launch: a grid has fewer than 2^32 threads, 256 to a workgroup here.
constexpr int64_t MAX_GRID = ((int64_t)1 << 24) - 1;

// No C++ exception crosses the ABI: a message that could not be built is the only one there is.
template <typename F>
int32_t guarded(F&& f) {
    try {
        return f();
    } catch (...) {
        return LLMDOT_E_NOMEM;
    }
}

// KvCache write and read: the same arguments and checks.
template <typename T, typename Launch>
int32_t move_rows(llmdot_hip_kv_cache* cache, T* k, int64_t ks, T* v, int64_t vs, const llmdot_hip_token_batch* batch,
                  const char* what, Launch launch) {
    if (!cache) return ctx_fail(LLMDOT_E_INVALID, "null cache");
    KvRows rows;
    int64_t total;
    if (int rc = check_rows(batch, &rows, &total)) return rc;
    const int64_t width = (int64_t)cache->view.kv_heads * cache->view.head_dim;
    if (int rc = check_stride("k", width, &ks)) return rc;
    if (int rc = check_stride("v", width, &vs)) return rc;
    if (total == 0) return 0;
    if (int rc = check_array("k", k)) return rc;
    if (int rc = check_array("v", v)) return rc;
    if (total * cache->view.kv_heads > MAX_GRID) return ctx_fail(LLMDOT_E_UNSUPPORTED, "too many rows in a call");
    OnDevice dev(ctx_device(cache->ctx));
    hipError_t e = dev.err;
    if (e == hipSuccess) e = launch(cache->view, rows, k, ks, v, vs, ctx_stream(cache->ctx));
    return e == hipSuccess ? 0 : device_error(what, e);
}

}  // namespace

extern "C" int32_t llmdot_hip_stream(llmdot_hip_ctx* ctx, void** stream) {
    if (!ctx || !stream) return ctx_fail(LLMDOT_E_INVALID, "null argument");
    *stream = ctx_stream(ctx);
    return 0;
}

extern "C" int32_t llmdot_hip_kv_cache_create(llmdot_hip_ctx* ctx, const llmdot_hip_kv_cache_desc* desc,
                                              llmdot_hip_kv_cache** out) {
    return guarded([&]() -> int32_t {
        if (!ctx || !desc || !out) return ctx_fail(LLMDOT_E_INVALID, "null argument");
        *out = nullptr;
        const auto& d = *desc;
        if (d.slots <= 0 || d.kv_heads <= 0 || d.head_dim <= 0 || d.capacity <= 0)
            return ctx_fail(LLMDOT_E_INVALID, "invalid KV cache description");
        if (!kv_attention_supported(d.head_dim))
            return ctx_fail(LLMDOT_E_UNSUPPORTED, "KV cache head_dim must be 64, 96, 128 or 256");
        if (d.capacity > (1 << 30)) return ctx_fail(LLMDOT_E_UNSUPPORTED, "KV cache capacity past 2^30 positions");
        for (uint32_t t : {d.k_type, d.v_type})
            if (t != GGML_Q8_0 && t != GGML_Q4_0)
                return ctx_fail(LLMDOT_E_UNSUPPORTED, "KV cache type " + std::to_string(t) + " is not Q8_0 or Q4_0");
        KvView v = kv_view(d.slots, d.kv_heads, d.head_dim, d.capacity, d.k_type == GGML_Q4_0, d.v_type == GGML_Q4_0);
        const double records = (double)d.slots * d.kv_heads * v.groups;
        if (records * (v.k_rec + v.v_rec) > 1e15) return ctx_fail(LLMDOT_E_NOMEM, "KV cache too large");
        const size_t kb = (size_t)records * v.k_rec, vb = (size_t)records * v.v_rec;
        OnDevice dev(ctx_device(ctx));
        if (dev.err != hipSuccess) return device_error("hipSetDevice", dev.err);
        auto* c = new (std::nothrow) llmdot_hip_kv_cache();
        if (!c) return ctx_fail(LLMDOT_E_NOMEM, "out of host memory");
        if (!ctx_hold(ctx)) {
            delete c;
            return ctx_fail(LLMDOT_E_INVALID, "the context has been destroyed");
        }
        // K and V in one allocation, zeroed on the stream that will read it
        hipError_t e = hipMalloc((void**)&v.k, kb + vb);
        if (e != hipSuccess) {
            (void)hipGetLastError();
            delete c;
            ctx_drop(ctx);
            return ctx_fail(LLMDOT_E_NOMEM, "KV cache of " + std::to_string(kb + vb) + " bytes: " + hipGetErrorString(e));
        }
        v.v = v.k + kb;
        e = hipMemsetAsync(v.k, 0, kb + vb, ctx_stream(ctx));
        if (e == hipSuccess) e = hipStreamSynchronize(ctx_stream(ctx));
        if (e != hipSuccess) {
            (void)hipFree(v.k);
            delete c;
            ctx_drop(ctx);
            return device_error("KV cache", e);
        }
        c->ctx = ctx;
        c->view = v;
        *out = c;
        return 0;
    });
}

extern "C" int32_t llmdot_hip_kv_cache_destroy(llmdot_hip_kv_cache* cache) {
    if (!cache) return 0;
    llmdot_hip_ctx* ctx = cache->ctx;
    {
        OnDevice dev(ctx_device(ctx));
        (void)hipStreamSynchronize(ctx_stream(ctx));
        (void)hipFree(cache->view.k);
    }
    delete cache;
    ctx_drop(ctx);
    return 0;
}

extern "C" int32_t llmdot_hip_kv_cache_write(llmdot_hip_kv_cache* cache, const float* k_dev, int64_t k_stride,
                                             const float* v_dev, int64_t v_stride,
                                             const llmdot_hip_token_batch* rows) {
    return guarded([&] { return move_rows(cache, k_dev, k_stride, v_dev, v_stride, rows, "kv_cache_write", launch_kv_write); });
}

extern "C" int32_t llmdot_hip_kv_cache_read(llmdot_hip_kv_cache* cache, float* k_dev, int64_t k_stride, float* v_dev,
                                            int64_t v_stride, const llmdot_hip_token_batch* rows) {
    return guarded([&] { return move_rows(cache, k_dev, k_stride, v_dev, v_stride, rows, "kv_cache_read", launch_kv_read); });
}

namespace {
int check_attention_shape(const llmdot_hip_kv_cache* cache, int heads, int64_t rows) {
    if (heads <= 0 || heads % cache->view.kv_heads != 0)
        return ctx_fail(LLMDOT_E_INVALID, "heads must be a multiple of the cache's kv_heads");
    if (rows * heads > MAX_GRID) return ctx_fail(LLMDOT_E_UNSUPPORTED, "too many rows in a call");
    return 0;
}
}  // namespace

extern "C" int32_t llmdot_hip_kv_cache_attention_workspace(const llmdot_hip_kv_cache* cache, int32_t heads, int32_t batch,
                                                           int32_t tokens, int32_t has_prefix, size_t* bytes) {
    return guarded([&]() -> int32_t {
        if (!cache || !bytes) return ctx_fail(LLMDOT_E_INVALID, "null argument");
        if (batch < 0 || tokens < 0) return ctx_fail(LLMDOT_E_INVALID, "negative batch or tokens");
        if (batch > MAX_SEQUENCES) return ctx_fail(LLMDOT_E_UNSUPPORTED, "more than 4096 sequences in a call");
        if (int rc = check_attention_shape(cache, heads, (int64_t)batch * tokens)) return rc;
        *bytes = batch && tokens ? kv_attention_workspace(cache->view, heads, batch, tokens, has_prefix != 0) : 0;
        return 0;
    });
}

extern "C" int32_t llmdot_hip_kv_cache_attention(llmdot_hip_kv_cache* cache, const float* q_dev, float* out_dev,
                                                 const llmdot_hip_token_batch* rows, const llmdot_hip_attention* opt,
                                                 void* workspace_dev, size_t workspace_bytes) {
    return guarded([&]() -> int32_t {
        if (!cache || !opt) return ctx_fail(LLMDOT_E_INVALID, "null argument");
        KvAttnArgs a{};
        int64_t total;
        if (int rc = check_rows(rows, &a.rows, &total)) return rc;
        if (int rc = check_attention_shape(cache, opt->heads, total)) return rc;
        const KvView& v = cache->view;
        const int64_t width = (int64_t)opt->heads * v.head_dim;
        a.q_stride = opt->q_stride; a.out_stride = opt->out_stride;
        if (int rc = check_stride("q", width, &a.q_stride)) return rc;
        if (int rc = check_stride("out", width, &a.out_stride)) return rc;
        if (opt->window < 0) return ctx_fail(LLMDOT_E_INVALID, "negative window");
        if (!(opt->scale >= 0.f) || opt->scale > 2e38f) return ctx_fail(LLMDOT_E_INVALID, "scale must be a number of at least 0");
        if (opt->prefix_len < 0) return ctx_fail(LLMDOT_E_INVALID, "negative prefix length");
        if (opt->prefix_len > 0 && !opt->prefix) return ctx_fail(LLMDOT_E_INVALID, "a prefix length without a prefix");
        if (opt->prefix && opt->prefix_len > 0) {
            const KvView& p = opt->prefix->view;
            if (opt->prefix->ctx != cache->ctx) return ctx_fail(LLMDOT_E_INVALID, "the prefix is of another context");
            if (p.kv_heads != v.kv_heads || p.head_dim != v.head_dim || p.k_q4 != v.k_q4 || p.v_q4 != v.v_q4)
                return ctx_fail(LLMDOT_E_INVALID, "the prefix has another shape or type");
            if (opt->prefix_slot < 0 || opt->prefix_slot >= p.slots || opt->prefix_len > p.capacity)
                return ctx_fail(LLMDOT_E_RANGE, "prefix slot or length outside its cache");
            a.prefix = p; a.prefix_slot = opt->prefix_slot; a.prefix_len = opt->prefix_len;
        }
        if (total == 0) return 0;
        if (int rc = check_array("q", q_dev)) return rc;
        if (int rc = check_array("out", out_dev)) return rc;
        const size_t need = kv_attention_workspace(v, opt->heads, a.rows.batch, a.rows.tokens, a.prefix_len > 0);
        if (need > 0) {
            if (int rc = check_array("workspace", workspace_dev)) return rc;
            if (workspace_bytes < need)
                return ctx_fail(LLMDOT_E_INVALID, "workspace of " + std::to_string(workspace_bytes) + " bytes, needs " +
                                                      std::to_string(need));
        }
        a.cache = v;
        a.q = q_dev; a.out = out_dev;
        a.heads = opt->heads; a.window = opt->window;
        a.scale = opt->scale > 0.f ? opt->scale : 1.0f / sqrtf((float)v.head_dim);
        a.work = static_cast<uint8_t*>(workspace_dev);
        OnDevice dev(ctx_device(cache->ctx));
        hipError_t e = dev.err;
        if (e == hipSuccess) e = launch_kv_attention(a, ctx_stream(cache->ctx));
        return e == hipSuccess ? 0 : device_error("kv_cache_attention", e);
    });
}

namespace {
int check_verify_shape(int batch, int drafts, int vocab) {
    if (batch < 0 || drafts < 0 || vocab <= 0) return ctx_fail(LLMDOT_E_INVALID, "bad batch, drafts or vocabulary");
    if (batch > MAX_SEQUENCES || drafts > 1024 || vocab > (1 << 24))
        return ctx_fail(LLMDOT_E_UNSUPPORTED, "at most 4096 sequences, 1024 drafts and 2^24 tokens in a vocabulary");
    if ((int64_t)batch * (vocab / 1024 + 1) > MAX_GRID) return ctx_fail(LLMDOT_E_UNSUPPORTED, "too many logits in a call");
    return 0;
}
}  // namespace

extern "C" int32_t llmdot_hip_verify_drafts_workspace(llmdot_hip_ctx* ctx, int32_t batch, int32_t drafts, int32_t vocab,
                                                      size_t* bytes) {
    return guarded([&]() -> int32_t {
        if (!ctx || !bytes) return ctx_fail(LLMDOT_E_INVALID, "null argument");
        if (int rc = check_verify_shape(batch, drafts, vocab)) return rc;
        *bytes = batch ? verify_workspace(batch, drafts, vocab) : 0;
        return 0;
    });
}

extern "C" int32_t llmdot_hip_verify_drafts(llmdot_hip_ctx* ctx, const float* target_dev, const float* draft_dev,
                                            const int32_t* drafts_dev, const int32_t* counts_dev,
                                            const float* uniforms_dev, int32_t batch, int32_t drafts, int32_t vocab,
                                            float temperature, int32_t* tokens_dev, int32_t* accepted_dev,
                                            void* workspace_dev, size_t workspace_bytes) {
    return guarded([&]() -> int32_t {
        if (!ctx) return ctx_fail(LLMDOT_E_INVALID, "null ctx");
        if (int rc = check_verify_shape(batch, drafts, vocab)) return rc;
        if (!(temperature <= 3e38f)) return ctx_fail(LLMDOT_E_INVALID, "temperature must be a number");
        if (batch == 0) return 0;
        if (int rc = check_array("target", target_dev)) return rc;
        if (draft_dev && !aligned(draft_dev)) return ctx_fail(LLMDOT_E_INVALID, "draft is not 16-byte aligned");
        if ((drafts > 0 && !drafts_dev) || !uniforms_dev || !tokens_dev || !accepted_dev)
            return ctx_fail(LLMDOT_E_INVALID, "null argument");
        const size_t need = verify_workspace(batch, drafts, vocab);
        if (need > 0) {
            if (int rc = check_array("workspace", workspace_dev)) return rc;
            if (workspace_bytes < need)
                return ctx_fail(LLMDOT_E_INVALID, "workspace of " + std::to_string(workspace_bytes) + " bytes, needs " +
                                                      std::to_string(need));
        }
        VerifyArgs a{target_dev, draft_dev, drafts_dev, counts_dev, uniforms_dev, batch, drafts, vocab, temperature,
                     tokens_dev, accepted_dev, static_cast<uint8_t*>(workspace_dev), 0.0, 0.0};
        OnDevice dev(ctx_device(ctx));
        hipError_t e = dev.err;
        if (e == hipSuccess) e = launch_verify(a, ctx_stream(ctx));
        return e == hipSuccess ? 0 : device_error("verify_drafts", e);
    });
}

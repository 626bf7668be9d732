// C entries of the 8-bit key/value cache (include/owk_kv8.h): argument checks, the device of the call,
// error reports. The kernels are in k_kv8.hip.
#include <cmath>
#include <cstdarg>

#include "kv8.h"

namespace owk {
namespace {

thread_local char g_kv8_error[256] = "";

int invalid(const char * fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_kv8_error, sizeof(g_kv8_error), fmt, ap);
    va_end(ap);
    return OWK_KV8_INVALID;
}

bool aligned(const void * p, size_t n) { return ((uintptr_t) p & (n - 1)) == 0; }

constexpr int kMaxGridYZ = 65535;  // entries and heads are grid dimensions

// the cache's description; 0 or the error
int check_cache(const owk_kv8_cache * c) {
    if (!c) return invalid("no cache");
    if (c->dtype != OWK_KV8_F16 && c->dtype != OWK_KV8_BF16) return invalid("cache dtype %d is neither f16 nor bf16", c->dtype);
    if (c->head_dim != 64 && c->head_dim != 128) return invalid("head_dim %d: 64 or 128 are supported", c->head_dim);
    if (c->n_heads < 1 || c->n_heads > kMaxGridYZ / 2) return invalid("n_heads %d out of range", c->n_heads);
    if (c->n_seqs < 1 || c->n_blocks < 1 || c->max_blocks < 1)
        return invalid("an empty cache (%d sequences, %d blocks, %d a sequence)", c->n_seqs, c->n_blocks, c->max_blocks);
    if (c->max_blocks > (1 << 24)) return invalid("max_blocks %d: token positions would pass 30 bits", c->max_blocks);
    if (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->k_tail || !c->v_tail) return invalid("a cache tensor is missing");
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 16) || !aligned(c->v_scale, 16) ||
        !aligned(c->k_tail, 16) || !aligned(c->v_tail, 16))
        return invalid("cache tensors have to be 16-byte aligned");
    if (!aligned(c->table, 4)) return invalid("the table is not 4-byte aligned");
    if (!c->table && (int64_t) c->n_seqs * c->max_blocks > c->n_blocks)
        return invalid("without a table %d sequences of %d blocks need %lld blocks, the pool has %d", c->n_seqs, c->max_blocks,
                       (long long) c->n_seqs * c->max_blocks, c->n_blocks);
    return 0;
}

int check_batch(const owk_kv8_batch * b) {
    if (!b) return invalid("no batch");
    if (b->n < 0 || b->n > kMaxGridYZ) return invalid("%d entries: 0 to %d are supported", b->n, kMaxGridYZ);
    if (b->max_new < 0 || b->max_new > (1 << 22)) return invalid("max_new %d out of range", b->max_new);
    if (b->n == 0) return 0;
    if (!b->lens) return invalid("lens is missing");
    if (b->off && (b->rows < 0 || b->rows > (int64_t) 1 << 40)) return invalid("rows %lld out of range", (long long) b->rows);
    if (!aligned(b->lens, 4) || !aligned(b->seq, 4) || !aligned(b->off, 4) || !aligned(b->count, 4))
        return invalid("an index array is not 4-byte aligned");
    return 0;
}

int check_rows(const char * name, const owk_kv8_rows * r, int bytes, Kv8Rows & out) {
    if (!r || !r->data) return invalid("%s is missing", name);
    if (!aligned(r->data, bytes)) return invalid("%s is not aligned to its elements", name);
    const int64_t most = (int64_t) 1 << 40;
    if (r->entry < 0 || r->row < 0 || r->head < 0 || r->entry > most || r->row > most || r->head > most)
        return invalid("strides of %s out of range", name);
    out.p = (char *) r->data;
    out.entry = r->entry;
    out.row = r->row;
    out.head = r->head;
    const int64_t e = 16 / bytes;
    out.vec = aligned(r->data, 16) && r->entry % e == 0 && r->row % e == 0 && r->head % e == 0;
    return 0;
}

int check_attend(const owk_kv8_cache * c, const owk_kv8_attend_params * p) {
    if (!p) return invalid("no params");
    if (p->n_q_heads < 1 || p->n_q_heads > kMaxGridYZ || p->n_q_heads % c->n_heads)
        return invalid("%d query heads are no multiple of %d key/value heads", p->n_q_heads, c->n_heads);
    if (p->out_type != c->dtype && p->out_type != OWK_KV8_F32) return invalid("out_type %d: the cache's type or f32", p->out_type);
    if (p->max_len < 0) return invalid("max_len %d is negative", p->max_len);
    if (!std::isfinite(p->scale)) return invalid("scale is not finite");
    return 0;
}

int capacity(const owk_kv8_cache * c) { return c->max_blocks * OWK_KV8_BLOCK; }

Kv8Plan plan_of(const owk_kv8_cache * c, const owk_kv8_batch * b, const owk_kv8_attend_params * p) {
    const int len = p->max_len > 0 && p->max_len < capacity(c) ? p->max_len : capacity(c);
    return kv8_plan(Kv8Call{*c, *b}, p->n_q_heads / c->n_heads, len);
}

// runs f on the cache's device and puts the caller's device back
template <typename F> int on_device(int device, F && f) {
    int before = -1;
    if (hipGetDevice(&before) != hipSuccess) {
        (void) hipGetLastError();
        snprintf(g_kv8_error, sizeof(g_kv8_error), "no usable device");
        return OWK_KV8_HIP;
    }
    if (device != before && hipSetDevice(device) != hipSuccess) {
        (void) hipGetLastError();
        return invalid("device %d is not there", device);
    }
    int rc = 0;
    const bool clean = hipPeekAtLastError() == hipSuccess;  // an older error of the caller's stays the caller's
    try {
        f();
        if (clean) OWK_HIP_CHECK(hipGetLastError());
    } catch (const std::exception & e) {
        snprintf(g_kv8_error, sizeof(g_kv8_error), "%s", e.what());
        rc = OWK_KV8_HIP;
    }
    if (device != before) (void) hipSetDevice(before);
    return rc;
}

} // namespace
} // namespace owk

using namespace owk;

extern "C" {

const char * owk_kv8_error(void) { return g_kv8_error; }

void owk_debug_kv8_entry(const owk_kv8_cache * cache, const owk_kv8_batch * batch, int b, int64_t out[4]) {
    const Kv8Entry e = kv8_entry(Kv8Call{*cache, *batch}, b);
    out[0] = e.seq;
    out[1] = e.start;
    out[2] = e.n;
    out[3] = e.row0;
}

void owk_debug_kv8_set_many_rows(int rows) { kv8_set_many_rows(rows); }

int64_t owk_debug_kv8_page(const owk_kv8_cache * cache, int seq, int i) { return kv8_page(*cache, seq, i); }

int owk_kv8_append(const owk_kv8_cache * cache, const owk_kv8_batch * batch, const owk_kv8_rows * k, const owk_kv8_rows * v,
                   void * stream) {
    Kv8Rows kr, vr;
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_batch(batch)) return rc;
    if (batch->n == 0 || batch->max_new == 0 || (batch->off && batch->rows == 0)) return 0;
    if (int rc = check_rows("k", k, 2, kr)) return rc;
    if (int rc = check_rows("v", v, 2, vr)) return rc;
    return on_device(cache->device, [&] { kv8_append((hipStream_t) stream, Kv8Call{*cache, *batch}, kr, vr); });
}

size_t owk_kv8_attend_workspace(const owk_kv8_cache * cache, const owk_kv8_batch * batch, const owk_kv8_attend_params * params) {
    if (check_cache(cache) || check_batch(batch) || check_attend(cache, params)) return 0;
    if (batch->n == 0 || batch->max_new == 0) return 0;
    return plan_of(cache, batch, params).ws_bytes;
}

int owk_kv8_attend(const owk_kv8_cache * cache, const owk_kv8_batch * batch, const owk_kv8_attend_params * params,
                   const owk_kv8_rows * q, const owk_kv8_rows * out, void * workspace, size_t workspace_bytes, void * stream) {
    Kv8Attend a;
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_batch(batch)) return rc;
    if (int rc = check_attend(cache, params)) return rc;
    if (batch->n == 0 || batch->max_new == 0 || (batch->off && batch->rows == 0)) return 0;
    if (int rc = check_rows("q", q, 2, a.q)) return rc;
    if (int rc = check_rows("out", out, params->out_type == OWK_KV8_F32 ? 4 : 2, a.out)) return rc;
    const Kv8Plan plan = plan_of(cache, batch, params);
    if (!plan.fits)
        return invalid("%d entries of up to %d rows and %d heads over up to %d tokens are too much for one call", batch->n, batch->max_new,
                       params->n_q_heads, params->max_len > 0 ? params->max_len : capacity(cache));
    if (plan.ws_bytes > 0) {
        if (!workspace || workspace_bytes < plan.ws_bytes)
            return invalid("a workspace of %zu bytes is needed, %zu are there", plan.ws_bytes, workspace ? workspace_bytes : 0);
        if (!aligned(workspace, 16)) return invalid("the workspace is not 16-byte aligned");
    }
    a.group = params->n_q_heads / cache->n_heads;
    a.causal = params->causal != 0;
    a.splits = plan.splits;
    a.per = plan.per;
    a.tiles = plan.tiles;
    a.join = plan.join;
    a.scale = params->scale;
    a.ws = (float *) workspace;
    return on_device(cache->device,
                     [&] { kv8_attend((hipStream_t) stream, Kv8Call{*cache, *batch}, a, plan, params->out_type); });
}

int owk_kv8_read(const owk_kv8_cache * cache, int n, int max_tokens, const int32_t * lens, const int32_t * seq,
                 const int32_t * first, const owk_kv8_rows * k, const owk_kv8_rows * v, void * stream) {
    Kv8Rows kr, vr;
    owk_kv8_batch b{};
    b.n = n;
    b.max_new = max_tokens;
    b.lens = lens;
    b.seq = seq;
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_batch(&b)) return rc;
    if (!aligned(first, 4)) return invalid("an index array is not 4-byte aligned");
    if (n == 0 || max_tokens == 0) return 0;
    if (int rc = check_rows("k", k, 2, kr)) return rc;
    if (int rc = check_rows("v", v, 2, vr)) return rc;
    return on_device(cache->device, [&] { kv8_read((hipStream_t) stream, Kv8Call{*cache, b}, first, kr, vr); });
}

} // extern "C"

// kvq8_api.cpp -- C ABI of the paged 8-bit key/value cache (hipgpt_attn.h):
// checks of arguments, then the launches of kvq8_cache.hip / kvq8_attn.hip.
#include <cmath>

#include "../../include/hipgpt_attn.h"
#include "kernels.h"
#include "kvq8.h"

using namespace hipgpt;

namespace {

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
int from_hip(hipError_t e) { return e == hipSuccess ? HIPGPT_OK : HIPGPT_ERR_LAUNCH; }
bool is_dtype(int t) { return t == HIPGPT_F32 || t == HIPGPT_BF16; }
// 16-byte rows of a [rows][heads][D] buffer
bool rows16(const void* p, int64_t ts, int64_t hs, int dtype) {
    const int64_t n = dtype == HIPGPT_F32 ? 4 : 8;
    return aligned(p, 16) && ts % n == 0 && hs % n == 0;
}

// (n - 1) * stride, n > 0 and stride > 0, at most 2^62
int64_t spread(int64_t n, int64_t stride) {
    const int64_t most = (int64_t)1 << 62;
    return n > 1 && stride > most / (n - 1) ? most : (n - 1) * stride;
}

// The cache and batch as the kernels take them; T: rows of the packed buffers.
int problem(const hipgpt_kvq8_cache* c, const hipgpt_kvq8_batch* b, int T, kvq8::Cache& out) {
    if (!c || !b || !c->k || !c->v || !c->k_scale || !c->v_scale || !b->block_table || !b->lens)
        return HIPGPT_ERR_INVALID;
    if (c->num_pages <= 0 || c->heads <= 0 || c->head_dim <= 0 || c->page_size <= 0 || b->batch <= 0 ||
        b->max_pages <= 0 || b->max_new <= 0 || T <= 0 || b->table_stride < 0 ||
        (b->batch > 1 && b->table_stride < b->max_pages))
        return HIPGPT_ERR_INVALID;
    if (!b->cu_new && (b->max_new != 1 || T != b->batch)) return HIPGPT_ERR_INVALID;
    if (!kvq8::supported(c->head_dim, c->page_size)) return HIPGPT_ERR_UNSUPPORTED;
    const int64_t bytes = (int64_t)c->page_size * c->head_dim;
    if (c->head_stride < bytes || c->page_stride < bytes || c->scale_page_stride < 1 || c->scale_head_stride < 1)
        return HIPGPT_ERR_INVALID;
    // pages and heads apart: heads inside a page's stride, or pages inside a head's
    if (c->page_stride < spread(c->heads, c->head_stride) + bytes &&
        c->head_stride < spread(c->num_pages, c->page_stride) + bytes)
        return HIPGPT_ERR_INVALID;
    if (c->scale_page_stride < spread(c->heads, c->scale_head_stride) + 1 &&
        c->scale_head_stride < spread(c->num_pages, c->scale_page_stride) + 1)
        return HIPGPT_ERR_INVALID;
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || c->page_stride % 16 || c->head_stride % 16)
        return HIPGPT_ERR_UNSUPPORTED;
    out.k = c->k;
    out.v = c->v;
    out.ks = c->k_scale;
    out.vs = c->v_scale;
    out.page_stride = c->page_stride;
    out.head_stride = c->head_stride;
    out.s_page_stride = c->scale_page_stride;
    out.s_head_stride = c->scale_head_stride;
    out.num_pages = c->num_pages;
    out.lps = c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
    out.H = c->heads;
    out.D = c->head_dim;
    out.table = b->block_table;
    out.t_stride = b->table_stride;
    out.max_pages = b->max_pages;
    out.lens = b->lens;
    out.cu = b->cu_new;
    out.B = b->batch;
    out.T = T;
    out.max_new = b->max_new < T ? b->max_new : T;
    return HIPGPT_OK;
}

// Both attention entry points.
int attention(const hipgpt_kvq8_cache* c, const hipgpt_kvq8_batch* b, int T, const void* q, void* o, int Hq,
              int64_t q_ts, int64_t q_hs, int64_t o_ts, int64_t o_hs, float scale, int dtype, int out_dtype,
              int num_splits, void* ws, size_t ws_bytes, hipStream_t stream) {
    kvq8::Cache k{};
    const int rc = problem(c, b, T, k);
    if (rc != HIPGPT_OK) return rc;
    if (!q || !o || Hq <= 0 || Hq % k.H != 0 || !std::isfinite(scale) || !is_dtype(dtype) || !is_dtype(out_dtype))
        return HIPGPT_ERR_INVALID;
    if (dtype == HIPGPT_F32 && out_dtype == HIPGPT_BF16) return HIPGPT_ERR_UNSUPPORTED;
    if ((int64_t)k.max_new * (Hq / k.H) > (1 << 30)) return HIPGPT_ERR_UNSUPPORTED;  // rows of one cached head
    if (!rows16(q, q_ts, q_hs, dtype) || !rows16(o, o_ts, o_hs, out_dtype)) return HIPGPT_ERR_UNSUPPORTED;
    const int64_t cap = (int64_t)k.max_pages << k.lps;
    int ns = num_splits > 0 ? num_splits
                            : kvq8::attn_splits(k.B, k.T, k.max_new, Hq, k.H, k.D, out_dtype,
                                                cap > 0x7fffffff ? 0x7fffffff : (int)cap);
    if (ns > kvq8::kMaxSplits) ns = kvq8::kMaxSplits;
    const size_t need = kvq8::attn_workspace(k.B, k.T, k.max_new, Hq, k.H, k.D, out_dtype, ns);
    if (need > 0 && (!ws || ws_bytes < need)) return HIPGPT_ERR_WORKSPACE;
    if (need > 0 && !aligned(ws, 16)) return HIPGPT_ERR_UNSUPPORTED;
    kvq8::AttnArgsQ8 a{};
    a.q = q;
    a.o = o;
    a.q_ts = q_ts;
    a.q_hs = q_hs;
    a.o_ts = o_ts;
    a.o_hs = o_hs;
    a.Hq = Hq;
    a.qscale = (scale > 0.f ? scale : 1.0f / std::sqrt((float)k.D)) * kLog2e;
    a.nsplit = ns;
    a.ws = static_cast<float*>(ws);
    return from_hip(kvq8::launch_attn(k, a, dtype, out_dtype, stream));
}

}  // namespace

extern "C" {

int hipgpt_rope_freqs(uint64_t* freqs, int rot_dim, double base) {
    if (!freqs || rot_dim <= 0 || rot_dim % 2 || !(base >= 1.0) || !std::isfinite(base)) return HIPGPT_ERR_INVALID;
    for (int i = 0; i < rot_dim / 2; ++i) {
        const long double turns = std::pow((long double)base, -2.0L * i / rot_dim) / 6.283185307179586476925286766559L;
        freqs[i] = (uint64_t)std::llrint(turns * 18446744073709551616.0L);
    }
    return HIPGPT_OK;
}

int hipgpt_kvq8_append(const hipgpt_kvq8_cache* cache, const hipgpt_kvq8_batch* batch, int T, const void* q,
                       void* q_out, const void* k, const void* v, int Hq, int64_t q_ts, int64_t q_hs, int64_t qo_ts,
                       int64_t qo_hs, int64_t k_ts, int64_t k_hs, int64_t v_ts, int64_t v_hs, const uint64_t* freqs,
                       int rot_dim, int interleaved, int dtype, int advance, hipStream_t stream) {
    if (!k || !v || !is_dtype(dtype) || (!q != !q_out) || (q && Hq <= 0)) return HIPGPT_ERR_INVALID;
    kvq8::Cache c{};
    const int rc = problem(cache, batch, T, c);
    if (rc != HIPGPT_OK) return rc;
    if (freqs && (rot_dim <= 0 || rot_dim % 2 || rot_dim > c.D)) return HIPGPT_ERR_INVALID;
    if (!rows16(k, k_ts, k_hs, dtype) || !rows16(v, v_ts, v_hs, dtype) ||
        (q && (!rows16(q, q_ts, q_hs, dtype) || !rows16(q_out, qo_ts, qo_hs, dtype))))
        return HIPGPT_ERR_UNSUPPORTED;
    kvq8::AppendArgs a{};
    a.q = q;
    a.q_out = q_out;
    a.k = k;
    a.v = v;
    a.q_ts = q_ts;
    a.q_hs = q_hs;
    a.qo_ts = qo_ts;
    a.qo_hs = qo_hs;
    a.k_ts = k_ts;
    a.k_hs = k_hs;
    a.v_ts = v_ts;
    a.v_hs = v_hs;
    a.Hq = Hq;
    a.freqs = freqs;
    a.rot = freqs ? rot_dim : 0;
    a.interleaved = interleaved ? 1 : 0;
    if (advance) {
        const int e = from_hip(kvq8::launch_advance(const_cast<int*>(c.lens), c.cu, c.B, stream));
        if (e != HIPGPT_OK) return e;
    }
    return from_hip(kvq8::launch_append(c, a, dtype, stream));
}

int hipgpt_kvq8_read(const hipgpt_kvq8_cache* cache, const hipgpt_kvq8_batch* batch, int T, void* k, void* v,
                     int64_t k_ts, int64_t k_hs, int64_t v_ts, int64_t v_hs, int dtype, hipStream_t stream) {
    if (!k || !v || !is_dtype(dtype)) return HIPGPT_ERR_INVALID;
    kvq8::Cache c{};
    const int rc = problem(cache, batch, T, c);
    if (rc != HIPGPT_OK) return rc;
    if (!rows16(k, k_ts, k_hs, dtype) || !rows16(v, v_ts, v_hs, dtype)) return HIPGPT_ERR_UNSUPPORTED;
    kvq8::ReadArgs a{};
    a.k = k;
    a.v = v;
    a.k_ts = k_ts;
    a.k_hs = k_hs;
    a.v_ts = v_ts;
    a.v_hs = v_hs;
    return from_hip(kvq8::launch_read(c, a, dtype, stream));
}

int hipgpt_attn_kvq8_default_splits(int B, int T, int max_new, int Hq, int heads, int D, int out_dtype, int max_len) {
    if (B <= 0 || T <= 0 || max_new <= 0 || Hq <= 0 || heads <= 0 || Hq % heads != 0 || D <= 0 || max_len <= 0)
        return 1;
    return kvq8::attn_splits(B, T, max_new < T ? max_new : T, Hq, heads, D, out_dtype, max_len);
}

size_t hipgpt_attn_kvq8_workspace_bytes(int B, int T, int max_new, int Hq, int heads, int D, int out_dtype,
                                        int num_splits) {
    if (B <= 0 || T <= 0 || max_new <= 0 || Hq <= 0 || heads <= 0 || Hq % heads != 0 || D <= 0) return 0;
    return kvq8::attn_workspace(B, T, max_new < T ? max_new : T, Hq, heads, D, out_dtype,
                                num_splits < kvq8::kMaxSplits ? num_splits : kvq8::kMaxSplits);
}

int hipgpt_attn_decode_kvq8(const hipgpt_kvq8_cache* cache, const hipgpt_kvq8_batch* batch, const void* q, void* o,
                            int Hq, int64_t q_ts, int64_t q_hs, int64_t o_ts, int64_t o_hs, float scale, int dtype,
                            int out_dtype, int num_splits, void* workspace, size_t workspace_bytes,
                            hipStream_t stream) {
    if (!batch || batch->cu_new || batch->max_new != 1) return HIPGPT_ERR_INVALID;
    return attention(cache, batch, batch->batch, q, o, Hq, q_ts, q_hs, o_ts, o_hs, scale, dtype, out_dtype, num_splits,
                     workspace, workspace_bytes, stream);
}

int hipgpt_attn_prefill_kvq8(const hipgpt_kvq8_cache* cache, const hipgpt_kvq8_batch* batch, int T, const void* q,
                             void* o, int Hq, int64_t q_ts, int64_t q_hs, int64_t o_ts, int64_t o_hs, float scale,
                             int dtype, int out_dtype, int num_splits, void* workspace, size_t workspace_bytes,
                             hipStream_t stream) {
    return attention(cache, batch, T, q, o, Hq, q_ts, q_hs, o_ts, o_hs, scale, dtype, out_dtype, num_splits, workspace,
                     workspace_bytes, stream);
}

}  // extern "C"

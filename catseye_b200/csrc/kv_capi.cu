// kv_capi.cu — C entry points of the paged Q4_0 KV cache and of the scoring
// of logits (include/catsgpu.h): checks of the arguments, then the launchers
// of kv.cu and score.cu.
#include "../../include/catsgpu.h"
#include "kv_pages.cuh"
#include "score.cuh"
#include <climits>
#include <new>

namespace cats {
int capi_fail(int code, const char *what);   // capi.cu
int capi_ready();
int capi_check(cudaError_t e, const char *what);
int *capi_err_word();
int capi_device();
cudaStream_t capi_stream();
}

using namespace cats;

static_assert(CATS_KV_PAGE == KV_PAGE && CATS_TYPE_F16 == KV_F16 && CATS_TYPE_BF16 == KV_BF16, "catsgpu.h");

struct cats_gpu_kv_pages {
    KvPages p;
};

namespace {

// Launches go to the library's device, whichever is current for the caller.
struct OnDevice {
    int was = -1;
    OnDevice()
    {
        int now = 0;
        if (cudaGetDevice(&now) == cudaSuccess && now != capi_device() && cudaSetDevice(capi_device()) == cudaSuccess)
            was = now;
    }
    ~OnDevice()
    {
        if (was >= 0) cudaSetDevice(was);
    }
};

size_t type_size(int type)
{
    return type == CATS_TYPE_F32 ? 4 : type == CATS_TYPE_F16 || type == CATS_TYPE_BF16 ? 2 : 0;
}

bool view_of(const cats_gpu_kv *c, int layer, KvView *v)
{
    if (!c || !c->pool || ((uintptr_t)c->pool % 16) || c->n_pages <= 0 || c->n_layers <= 0 || c->n_kv_heads <= 0 ||
        layer < 0 || layer >= c->n_layers || c->head_size <= 0 || c->head_size % 32 || c->head_size > KV_MAX_HS)
        return false;
    const size_t layer_bytes = (size_t)c->n_kv_heads * 72 * c->head_size;
    v->pool = static_cast<uint8_t *>(c->pool) + layer * layer_bytes;
    v->page_bytes = layer_bytes * c->n_layers;
    v->table = c->table;
    v->n_pages = c->n_pages;
    v->n_kv = c->n_kv_heads;
    v->hs = c->head_size;
    v->n_seqs = c->n_seqs;
    v->max_pages = c->max_pages;
    v->err = nullptr;
    return true;
}

bool tabled(const cats_gpu_kv *c)
{
    return c && c->table && c->n_seqs > 0 && c->max_pages > 0 && c->max_pages <= INT_MAX / KV_PAGE;
}

bool rows_ok(const void *p, int type, long long ld, int rows, long long width, KvRows *r)
{
    const size_t ts = type_size(type);
    if (!ts || !p || (uintptr_t)p % ts || rows <= 0 || ld < width) return false;
    *r = KvRows{const_cast<void *>(p), ld, rows, (uintptr_t)p % (4 * ts) == 0 && ld % 4 == 0};
    return true;
}

cudaStream_t on(void *stream) { return stream ? (cudaStream_t)stream : capi_stream(); }

int rows_call(const cats_gpu_kv *c, int layer, void *k, void *v, int type, long long ld_k, long long ld_v, int rows,
              const int *runs, int n_runs, int max_rows, void *stream, bool append, const char *what)
{
    if (c && c->head_size > KV_MAX_HS) return capi_fail(CATS_ERR_UNSUPPORTED, what);
    KvView view;
    KvRows rk, rv;
    if (rows == 0 || n_runs == 0) return CATS_OK;
    if (!tabled(c) || !view_of(c, layer, &view) || !runs || n_runs < 0 || max_rows < 0 || (!append && k == v) ||
        !rows_ok(k, type, ld_k, rows, (long long)c->n_kv_heads * c->head_size, &rk) ||
        !rows_ok(v, type, ld_v, rows, (long long)c->n_kv_heads * c->head_size, &rv))
        return capi_fail(CATS_ERR_ARG, what);
    if (int rc = capi_ready()) return rc;
    view.err = capi_err_word();
    OnDevice dev;
    const KvBatch b{reinterpret_cast<const KvRun *>(runs), n_runs, max_rows, 0};
    return capi_check((append ? launch_kv_append : launch_kv_read)(view, type, rk, rv, b, on(stream)), what);
}

} // namespace

extern "C" {

size_t cats_gpu_kv_page_bytes(int n_layers, int n_kv_heads, int head_size)
{
    if (n_layers <= 0 || n_kv_heads <= 0 || head_size <= 0 || head_size % 32 || head_size > KV_MAX_HS) return 0;
    return (size_t)n_layers * n_kv_heads * 72 * head_size;
}

int cats_gpu_kv_append_dev(const cats_gpu_kv *c, int layer, const void *k, const void *v, int type, long long ld_k,
                           long long ld_v, int rows, const int *runs, int n_runs, int max_rows, void *stream)
{
    return rows_call(c, layer, const_cast<void *>(k), const_cast<void *>(v), type, ld_k, ld_v, rows, runs, n_runs,
                     max_rows, stream, true, "cats_gpu_kv_append_dev");
}

int cats_gpu_kv_read_dev(const cats_gpu_kv *c, int layer, void *k, void *v, int type, long long ld_k, long long ld_v,
                         int rows, const int *runs, int n_runs, int max_rows, void *stream)
{
    return rows_call(c, layer, k, v, type, ld_k, ld_v, rows, runs, n_runs, max_rows, stream, false,
                     "cats_gpu_kv_read_dev");
}

int cats_gpu_kv_attention_dev(const cats_gpu_kv *c, int layer, void *out, const void *q, int type, int n_heads,
                              long long ld_out, long long ld_q, int rows, const int *runs, int n_runs, int max_rows,
                              int max_len, void *stream)
{
    const char *what = "cats_gpu_kv_attention_dev";
    if (c && c->head_size > KV_MAX_HS) return capi_fail(CATS_ERR_UNSUPPORTED, what);
    KvView view;
    KvRows rq, ro;
    if (rows == 0 || n_runs == 0) return CATS_OK;
    if (!tabled(c) || !view_of(c, layer, &view) || !runs || n_runs < 0 || max_rows < 0 || max_len < 0 || out == q ||
        n_heads <= 0 || n_heads % c->n_kv_heads ||
        !rows_ok(q, type, ld_q, rows, (long long)n_heads * c->head_size, &rq) ||
        !rows_ok(out, type, ld_out, rows, (long long)n_heads * c->head_size, &ro))
        return capi_fail(CATS_ERR_ARG, what);
    if (int rc = capi_ready()) return rc;
    view.err = capi_err_word();
    OnDevice dev;
    const KvBatch b{reinterpret_cast<const KvRun *>(runs), n_runs, max_rows, max_len};
    return capi_check(launch_kv_attention(view, type, ro, rq, n_heads, b, on(stream)), what);
}

int cats_gpu_kv_copy_pages_dev(const cats_gpu_kv *c, const int *src, const int *dst, int n, void *stream)
{
    const char *what = "cats_gpu_kv_copy_pages_dev";
    if (c && c->head_size > KV_MAX_HS) return capi_fail(CATS_ERR_UNSUPPORTED, what);
    KvView view;
    if (n == 0) return CATS_OK;
    if (!view_of(c, 0, &view) || !src || !dst || n < 0 || n > c->n_pages) return capi_fail(CATS_ERR_ARG, what);
    // every page is at most one copy's destination, and then no copy's source
    try {
        std::vector<uint8_t> is(c->n_pages, 0);
        for (int i = 0; i < n; i++) {
            if (src[i] < 0 || src[i] >= c->n_pages || dst[i] < 0 || dst[i] >= c->n_pages || is[dst[i]])
                return capi_fail(CATS_ERR_ARG, what);
            is[dst[i]] = 1;
        }
        for (int i = 0; i < n; i++)
            if (is[src[i]]) return capi_fail(CATS_ERR_ARG, what);
    } catch (const std::bad_alloc &) {
        return capi_fail(CATS_ERR_NOMEM, what);
    }
    if (int rc = capi_ready()) return rc;
    OnDevice dev;
    return capi_check(launch_kv_copy(view.pool, view.page_bytes, src, dst, n, on(stream)), what);
}

cats_gpu_kv_pages *cats_gpu_kv_pages_create(int n_pages, int n_seqs, int max_pages)
{
    if (n_pages <= 0 || n_seqs <= 0 || max_pages <= 0 || max_pages > INT_MAX / KV_PAGE) {
        capi_fail(CATS_ERR_ARG, "cats_gpu_kv_pages_create");
        return nullptr;
    }
    try {
        return new cats_gpu_kv_pages{KvPages(n_pages, n_seqs, max_pages)};
    } catch (const std::bad_alloc &) {
        capi_fail(CATS_ERR_NOMEM, "cats_gpu_kv_pages_create");
        return nullptr;
    }
}

void cats_gpu_kv_pages_destroy(cats_gpu_kv_pages *p) { delete p; }

// The copies an operation asks for, into the caller's arrays.
static int give(const std::vector<int> &s, const std::vector<int> &d, int *src, int *dst, int *n)
{
    for (size_t i = 0; i < s.size(); i++) {
        src[i] = s[i];
        dst[i] = d[i];
    }
    *n = (int)s.size();
    return CATS_OK;
}

int cats_gpu_kv_pages_write(cats_gpu_kv_pages *p, int seq, int pos, int n, int *src, int *dst, int *n_copies)
{
    const char *what = "cats_gpu_kv_pages_write";
    if (!p || !src || !dst || !n_copies) return capi_fail(CATS_ERR_ARG, what);
    try {
        std::vector<int> s, d;
        if (n > 0) { s.reserve(n / KV_PAGE + 2); d.reserve(n / KV_PAGE + 2); }
        if (int rc = p->p.write(seq, pos, n, s, d)) return capi_fail(rc, what);
        return give(s, d, src, dst, n_copies);
    } catch (const std::bad_alloc &) {
        return capi_fail(CATS_ERR_NOMEM, what);
    }
}

int cats_gpu_kv_pages_fork(cats_gpu_kv_pages *p, int src_seq, int dst_seq, int len)
{
    const char *what = "cats_gpu_kv_pages_fork";
    if (!p) return capi_fail(CATS_ERR_ARG, what);
    try {
        const int rc = p->p.fork(src_seq, dst_seq, len);
        return rc ? capi_fail(rc, what) : CATS_OK;
    } catch (const std::bad_alloc &) {
        return capi_fail(CATS_ERR_NOMEM, what);
    }
}

int cats_gpu_kv_pages_truncate(cats_gpu_kv_pages *p, int seq, int len)
{
    const char *what = "cats_gpu_kv_pages_truncate";
    if (!p) return capi_fail(CATS_ERR_ARG, what);
    try {
        const int rc = p->p.truncate(seq, len);
        return rc ? capi_fail(rc, what) : CATS_OK;
    } catch (const std::bad_alloc &) {
        return capi_fail(CATS_ERR_NOMEM, what);
    }
}

int cats_gpu_kv_pages_compact(cats_gpu_kv_pages *p, int *src, int *dst, int *n_copies)
{
    const char *what = "cats_gpu_kv_pages_compact";
    if (!p || !src || !dst || !n_copies) return capi_fail(CATS_ERR_ARG, what);
    try {
        std::vector<int> s, d;
        s.reserve(p->p.n_pages());
        d.reserve(p->p.n_pages());
        p->p.compact(s, d);
        return give(s, d, src, dst, n_copies);
    } catch (const std::bad_alloc &) {
        return capi_fail(CATS_ERR_NOMEM, what);
    }
}

int cats_gpu_kv_pages_length(const cats_gpu_kv_pages *p, int seq) { return p && p->p.seq_ok(seq) ? p->p.length(seq) : -1; }
int cats_gpu_kv_pages_free(const cats_gpu_kv_pages *p) { return p ? p->p.free_count() : -1; }
const int *cats_gpu_kv_pages_table(const cats_gpu_kv_pages *p) { return p ? p->p.table() : nullptr; }

int cats_gpu_logprobs_dev(const void *logits, int type, int rows, int vocab, long long ld, const int *targets, int k,
                          float *logprob, float *entropy, int *top_ids, float *top_logprob, void *stream)
{
    const char *what = "cats_gpu_logprobs_dev";
    if (k > SCORE_MAX_K) return capi_fail(CATS_ERR_UNSUPPORTED, what);
    if (rows == 0) return CATS_OK;
    const size_t ts = type_size(type);
    if (!ts || !logits || (uintptr_t)logits % ts || rows < 0 || vocab <= 0 || ld < vocab || k < 0 ||
        (logprob && !targets) || (k > 0 && (!top_ids || !top_logprob)))
        return capi_fail(CATS_ERR_ARG, what);
    if (int rc = capi_ready()) return rc;
    OnDevice dev;
    const ScoreArgs a{logits, targets, logprob, entropy, top_ids, top_logprob, ld, rows, vocab, k, capi_err_word()};
    return capi_check(launch_logprobs(a, type, on(stream)), what);
}

} // extern "C"

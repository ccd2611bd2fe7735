// kv_model.cu — the batched step on a paged Q4_0 cache (kv_model.cuh).
#include "kv_model.cuh"
#include <algorithm>
#include <cstring>
#include <new>
#include <utility>

namespace cats {

static void drop_graph(LlmModel *m)
{
    if (m->bt_exec) cudaGraphExecDestroy(m->bt_exec);
    if (m->bt_graph) cudaGraphDestroy(m->bt_graph);
    m->bt_exec = nullptr;
    m->bt_graph = nullptr;
    m->bt_graph_T = 0;
}

static void free_rows(LlmPaged *p)
{
    for (void *d : {(void *)p->runs, (void *)p->q16, (void *)p->o16})
        if (d) cudaFree(d);
    if (p->runs_host) cudaFreeHost(p->runs_host);
    p->runs = p->runs_host = nullptr;
    p->q16 = p->o16 = nullptr;
    p->cap = 0;
}

void llm_paged_free(LlmModel *m)
{
    LlmPaged *p = m->paged;
    if (!p) return;
    free_rows(p);
    if (p->pool) cudaFree(p->pool);
    if (p->table) cudaFree(p->table);
    if (p->table_host) cudaFreeHost(p->table_host);
    delete p;
    m->paged = nullptr;
}

int llm_cache_q4(LlmModel *m, int n_pages, int n_seqs)
{
    if (cudaStreamSynchronize(m->stream) != cudaSuccess) return E_CUDA;
    if (n_pages == 0) {
        drop_graph(m);
        llm_paged_free(m);
        return E_OK;
    }
    if (n_pages < 0 || n_seqs <= 0) return E_ARG;
    if (!batch_supported(m) || m->head_size % 32 || m->head_size > KV_MAX_HS) return E_UNSUPPORTED;
    const int max_pages = (m->c.seq_len + KV_PAGE - 1) / KV_PAGE;
    const size_t page_bytes = (size_t)m->c.n_layers * m->kv_heads_loc * 72 * m->head_size;
    size_t free_mem = 0, all = 0;   // (before the host's lists of so many pages are made)
    if (cudaMemGetInfo(&free_mem, &all) != cudaSuccess || all / page_bytes < (size_t)n_pages) return E_NOMEM;
    LlmPaged *p = nullptr;
    try {
        p = new LlmPaged(n_pages, n_seqs, max_pages);
        p->sent.assign((size_t)n_seqs * max_pages, -1);
    } catch (const std::bad_alloc &) {
        delete p;
        return E_NOMEM;
    }
    p->page_bytes = page_bytes;
    const size_t tb = (size_t)n_seqs * max_pages * 4;
    bool ok = cudaMalloc(&p->pool, p->page_bytes * n_pages) == cudaSuccess;
    ok = ok && cudaMalloc(&p->table, tb) == cudaSuccess && cudaMallocHost(&p->table_host, tb) == cudaSuccess;
    ok = ok && cudaMemset(p->table, 0xff, tb) == cudaSuccess;
    if (!ok) {
        cudaGetLastError();
        std::swap(m->paged, p);   // free the new one, keep what was there
        llm_paged_free(m);
        m->paged = p;
        return E_NOMEM;
    }
    drop_graph(m);
    llm_paged_free(m);
    m->paged = p;
    return E_OK;
}

KvView llm_paged_view(const LlmModel *m, int layer)
{
    const LlmPaged *p = m->paged;
    KvView v;
    v.pool = p->pool + (size_t)layer * m->kv_heads_loc * 72 * m->head_size;
    v.table = p->table;
    v.page_bytes = p->page_bytes;
    v.n_pages = p->pages.n_pages();
    v.n_kv = m->kv_heads_loc;
    v.hs = m->head_size;
    v.n_seqs = p->pages.n_seqs();
    v.max_pages = p->pages.max_pages();
    v.err = m->err;
    return v;
}

// The page copies an operation asked for, then the table.  The stream is idle
// (the callers synchronise it), so the pinned staging is free.
static int settle(LlmModel *m, const std::vector<int> &src, const std::vector<int> &dst)
{
    LlmPaged *p = m->paged;
    if (!src.empty() &&
        launch_kv_copy(p->pool, p->page_bytes, src.data(), dst.data(), (int)src.size(), m->stream) != cudaSuccess)
        return E_CUDA;
    const size_t tb = (size_t)p->pages.n_seqs() * p->pages.max_pages() * 4;
    memcpy(p->table_host, p->pages.table(), tb);
    memcpy(p->sent.data(), p->pages.table(), tb);
    return cudaMemcpyAsync(p->table, p->table_host, tb, cudaMemcpyHostToDevice, m->stream) == cudaSuccess ? E_OK : E_CUDA;
}

// A few entries of the table, as the kernel's parameters: no staging that an
// earlier copy may still read, so the host need not wait for the stream.
constexpr int KV_PATCH = 240;
struct KvPatch {
    unsigned long long at[KV_PATCH];
    int page[KV_PATCH];
};
__global__ void k_kv_patch(int *table, int n, const __grid_constant__ KvPatch p)
{
    if ((int)threadIdx.x < n) table[p.at[threadIdx.x]] = p.page[threadIdx.x];
}

// Positions of a sequence to make writable.
struct Stretch {
    int seq, pos, n;
};

// The page copies, and the entries of the stretches that changed, in stream order.
static int settle_behind(LlmModel *m, const std::vector<Stretch> &s, const std::vector<int> &src, const std::vector<int> &dst)
{
    LlmPaged *p = m->paged;
    if (!src.empty() &&
        launch_kv_copy(p->pool, p->page_bytes, src.data(), dst.data(), (int)src.size(), m->stream) != cudaSuccess)
        return E_CUDA;
    KvPatch patch;
    int n = 0;
    auto send = [&] {
        if (n > 0) k_kv_patch<<<1, 256, 0, m->stream>>>(p->table, n, patch);
        n = 0;
        return cudaGetLastError() == cudaSuccess;
    };
    for (const Stretch &x : s)
        for (int i = x.pos / KV_PAGE; x.n > 0 && i <= (x.pos + x.n - 1) / KV_PAGE; i++) {
            const size_t at = (size_t)x.seq * p->pages.max_pages() + i;
            if (p->sent[at] == p->pages.table()[at]) continue;
            patch.at[n] = at;
            patch.page[n++] = p->sent[at] = p->pages.table()[at];
            if (n == KV_PATCH && !send()) return E_CUDA;
        }
    return send() ? E_OK : E_CUDA;
}

// Make stretches writable, all of them or none; the
// device's table follows where it changed.  idle: nothing is enqueued on the
// stream.
static int write_all(LlmModel *m, std::vector<Stretch> s, bool idle)
{
    KvPages &pg = m->paged->pages;
    std::sort(s.begin(), s.end(), [](const Stretch &a, const Stretch &b) { return a.seq != b.seq ? a.seq < b.seq : a.pos < b.pos; });
    int end = 0;
    for (size_t i = 0; i < s.size(); i++) {
        if (i == 0 || s[i].seq != s[i - 1].seq) end = pg.length(s[i].seq);
        else if (s[i].pos < s[i - 1].pos + s[i - 1].n) return E_ARG;   // a position twice
        if (s[i].pos > end || (long long)s[i].pos + s[i].n > m->c.seq_len) return E_ARG;
        end = std::max(end, s[i].pos + s[i].n);
    }
    // The sum of the needs is an upper bound (two stretches may want the same
    // page); past it, try on a copy.
    long long need = 0;
    for (const Stretch &x : s) need += pg.need(x.seq, x.pos, x.n);
    std::vector<int> src, dst;
    src.reserve(need);
    dst.reserve(need);
    if (need > pg.free_count()) {
        KvPages trial = pg;
        for (const Stretch &x : s)
            if (int rc = trial.reserve(x.seq, x.pos, x.n, src, dst)) return rc;
        pg = std::move(trial);
    } else {
        for (const Stretch &x : s)
            if (int rc = pg.reserve(x.seq, x.pos, x.n, src, dst)) return rc;
    }
    if (!idle) return settle_behind(m, s, src, dst);
    const size_t tb = (size_t)pg.n_seqs() * pg.max_pages() * 4;
    return src.empty() && !memcmp(m->paged->sent.data(), pg.table(), tb) ? E_OK : settle(m, src, dst);
}

static int reserve_rows(LlmModel *m)
{
    LlmPaged *p = m->paged;
    if (p->cap >= m->bt_cap) return E_OK;
    drop_graph(m);
    free_rows(p);
    const size_t n = m->bt_cap;
    bool ok = cudaMalloc(&p->runs, n * sizeof(KvRun)) == cudaSuccess &&
              cudaMallocHost(&p->runs_host, n * sizeof(KvRun)) == cudaSuccess &&
              cudaMalloc(&p->q16, n * m->q_dim * 2) == cudaSuccess && cudaMalloc(&p->o16, n * m->q_dim * 2) == cudaSuccess;
    if (!ok) {
        cudaGetLastError();
        free_rows(p);
        return E_NOMEM;
    }
    p->cap = m->bt_cap;
    return E_OK;
}

int llm_paged_set(LlmModel *m, int T, int ahead)
try {
    LlmPaged *p = m->paged;
    if (int rc = reserve_rows(m)) return rc;
    const BatchTok *tok = m->bt_tok_host;
    std::vector<Stretch> s;
    int nr = 0, rows = 0, len = 0;
    for (int t = 0; t < T;) {
        int n = 1;
        while (t + n < T && tok[t + n].seq == tok[t].seq && tok[t + n].pos == tok[t].pos + n) n++;
        p->runs_host[nr++] = KvRun{t, n, tok[t].seq, tok[t].pos};
        s.push_back({tok[t].seq, tok[t].pos, ahead ? std::max(n, ahead) : 0});
        rows = std::max(rows, n);
        len = std::max(len, tok[t].pos + n);
        t += n;
    }
    for (int q : p->set_seqs) p->pages.truncate(q, p->pages.length(q));   // what never ran
    p->set_seqs.clear();
    for (const Stretch &x : s) p->set_seqs.push_back(x.seq);
    if (int rc = write_all(m, s, true)) return rc;
    p->n_runs = nr;
    p->max_rows = rows;
    p->max_len = len;
    p->advanced = 0;
    return cudaMemcpyAsync(p->runs, p->runs_host, (size_t)nr * sizeof(KvRun), cudaMemcpyHostToDevice, m->stream) == cudaSuccess
               ? E_OK : E_CUDA;
} catch (const std::bad_alloc &) {
    return E_NOMEM;
}

int llm_paged_extend(LlmModel *m, int T, int steps)
try {
    LlmPaged *p = m->paged;
    if (p->n_runs != T) return E_ARG;   // a run of several tokens is not a decode batch
    std::vector<Stretch> s;
    for (int t = 0; t < T; t++) s.push_back({m->bt_tok_host[t].seq, m->bt_tok_host[t].pos + p->advanced, steps});
    return write_all(m, s, false);
} catch (const std::bad_alloc &) {
    return E_NOMEM;
}

void llm_paged_count(LlmModel *m, int T, int steps, bool move)
{
    LlmPaged *p = m->paged;
    for (int t = 0; t < T; t++) p->pages.count(m->bt_tok_host[t].seq, m->bt_tok_host[t].pos + p->advanced + steps);
    if (move) p->advanced += steps;
}

int llm_cache_fork(LlmModel *m, int src, int dst, int len)
{
    if (cudaStreamSynchronize(m->stream) != cudaSuccess) return E_CUDA;
    const int rc = m->paged->pages.fork(src, dst, len);
    return rc ? rc : settle(m, {}, {});
}

int llm_cache_truncate(LlmModel *m, int seq, int len)
{
    if (cudaStreamSynchronize(m->stream) != cudaSuccess) return E_CUDA;
    const int rc = m->paged->pages.truncate(seq, len);
    return rc ? rc : settle(m, {}, {});
}

int llm_cache_compact(LlmModel *m, int *moved)
{
    if (cudaStreamSynchronize(m->stream) != cudaSuccess) return E_CUDA;
    std::vector<int> src, dst;
    m->paged->pages.compact(src, dst);
    if (moved) *moved = (int)src.size();
    return settle(m, src, dst);
}

// k, v: device rows [n][kv_dim] of one layer
static cudaError_t read_rows(LlmModel *m, int layer, int seq, int n, float *k, float *v, KvRun *d_run)
{
    const KvRun run{0, n, seq, 0};
    cudaError_t e = cudaMemcpyAsync(d_run, &run, sizeof run, cudaMemcpyHostToDevice, m->stream);
    if (e) return e;
    return launch_kv_read(llm_paged_view(m, layer), KV_F32, KvRows{k, m->kv_dim, n, 1}, KvRows{v, m->kv_dim, n, 1},
                          KvBatch{d_run, 1, n, n}, m->stream);
}

int llm_cache_read(LlmModel *m, int layer, int seq, int n, float *k_host, float *v_host)
{
    LlmPaged *p = m->paged;
    if (layer < 0 || layer >= m->c.n_layers || !p->pages.seq_ok(seq) || n < 0 || n > p->pages.length(seq)) return E_ARG;
    if (n == 0) return E_OK;
    const size_t bytes = (size_t)n * m->kv_dim * 4;
    uint8_t *d = nullptr;
    if (cudaMalloc(&d, 2 * bytes + sizeof(KvRun)) != cudaSuccess) {
        cudaGetLastError();
        return E_NOMEM;
    }
    float *k = reinterpret_cast<float *>(d), *v = k + (size_t)n * m->kv_dim;
    bool ok = read_rows(m, layer, seq, n, k, v, reinterpret_cast<KvRun *>(d + 2 * bytes)) == cudaSuccess;
    ok = ok && cudaMemcpyAsync(k_host, k, bytes, cudaMemcpyDeviceToHost, m->stream) == cudaSuccess &&
         cudaMemcpyAsync(v_host, v, bytes, cudaMemcpyDeviceToHost, m->stream) == cudaSuccess;
    ok = cudaStreamSynchronize(m->stream) == cudaSuccess && ok;
    cudaFree(d);
    return ok ? E_OK : E_CUDA;
}

int llm_cache_to_dense(LlmModel *m, int seq, int n)
{
    LlmPaged *p = m->paged;
    if (!p->pages.seq_ok(seq) || n < 0 || n > p->pages.length(seq)) return E_ARG;
    if (n == 0) return E_OK;
    KvRun *d = nullptr;
    if (cudaMalloc(&d, sizeof(KvRun)) != cudaSuccess) {
        cudaGetLastError();
        return E_NOMEM;
    }
    bool ok = true;
    for (int l = 0; l < m->c.n_layers && ok; l++) {
        const size_t at = (size_t)l * m->c.seq_len * m->kv_dim;
        ok = read_rows(m, l, seq, n, m->kcache + at, m->vcache + at, d) == cudaSuccess;
    }
    ok = cudaStreamSynchronize(m->stream) == cudaSuccess && ok;
    cudaFree(d);
    return ok ? E_OK : E_CUDA;
}

} // namespace cats

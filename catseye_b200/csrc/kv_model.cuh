// kv_model.cuh — the batched step's paged Q4_0 cache: the model's pages, the
// batch as runs, and what keeps both in step with the device.
#pragma once
#include "kv_pages.cuh"
#include "llm.cuh"

namespace cats {

struct LlmPaged {
    KvPages pages;
    size_t page_bytes = 0;
    uint8_t *pool = nullptr;               // device
    int *table = nullptr, *table_host = nullptr;   // device; pinned staging
    std::vector<int> sent;                 // what the device's table holds once the stream gets there
    KvRun *runs = nullptr, *runs_host = nullptr;
    __half *q16 = nullptr, *o16 = nullptr; // [cap][q_dim]: queries (RoPE applied) and attention output
    int cap = 0;                           // tokens runs / q16 / o16 hold
    int n_runs = 0, max_rows = 0, max_len = 0;
    int advanced = 0;                      // greedy steps enqueued since the batch was set
    std::vector<int> set_seqs;             // the set batch's sequences

    LlmPaged(int n_pages, int n_seqs, int max_pages) : pages(n_pages, n_seqs, max_pages) {}
};

// Switch the batched step to n_pages pages shared by n_seqs sequences (0
// pages: back to the dense cache).  E_UNSUPPORTED for head sizes the cache
// does not take.
int llm_cache_q4(LlmModel *m, int n_pages, int n_seqs);
void llm_paged_free(LlmModel *m);
// Group the batch in m->bt_tok_host into runs, make their positions writable
// (from each run's first, at least `ahead`; 0: none) and upload table and runs.
// The sequences' lengths stay: positions count once what writes them is
// enqueued (llm_paged_count), and the pages of a batch that never ran are free
// again when the next one is set.
int llm_paged_set(LlmModel *m, int T, int ahead);
// Make the next `steps` positions of a batch of single tokens writable, behind
// what is enqueued (the host does not wait).
int llm_paged_extend(LlmModel *m, int T, int steps);
// The batch's next `steps` positions a token are enqueued; move: the batch has
// moved on over them.
void llm_paged_count(LlmModel *m, int T, int steps, bool move);
KvView llm_paged_view(const LlmModel *m, int layer);
int llm_cache_fork(LlmModel *m, int src, int dst, int len);
int llm_cache_truncate(LlmModel *m, int seq, int len);
int llm_cache_compact(LlmModel *m, int *moved);
// Rows 0 .. n - 1 of a sequence: K and V [n][kv_dim] floats to host, or into
// the dense cache's sequence 0, which the single-token engines read.
int llm_cache_read(LlmModel *m, int layer, int seq, int n, float *k_host, float *v_host);
int llm_cache_to_dense(LlmModel *m, int seq, int n);

} // namespace cats

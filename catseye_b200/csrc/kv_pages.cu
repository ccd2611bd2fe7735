// kv_pages.cu — page bookkeeping of the paged KV cache (kv_pages.cuh).  Host
// code only: it runs without a GPU.
#include "kv_pages.cuh"
#include <algorithm>

namespace cats {

KvPages::KvPages(int n_pages, int n_seqs, int max_pages)
    : max_pages_(max_pages), table_((size_t)n_seqs * max_pages, -1), refs_(n_pages, 0), len_(n_seqs, 0)
{
    for (int i = 0; i < n_pages; i++) free_.insert(free_.end(), i);
}

int KvPages::take()
{
    const int p = *free_.begin();
    free_.erase(free_.begin());
    refs_[p] = 1;
    return p;
}

void KvPages::drop(int page)
{
    if (--refs_[page] == 0) free_.insert(page);
}

int KvPages::need(int seq, int pos, int n) const
{
    int k = 0;
    const int *t = row(seq);
    for (int i = pos / KV_PAGE; n > 0 && i <= (pos + n - 1) / KV_PAGE; i++) k += t[i] < 0 || refs_[t[i]] > 1;
    return k;
}

int KvPages::write(int seq, int pos, int n, std::vector<int> &src, std::vector<int> &dst)
{
    if (!seq_ok(seq) || pos > len_[seq]) return E_ARG;
    if (int rc = reserve(seq, pos, n, src, dst)) return rc;
    if (n > 0) count(seq, pos + n);
    return E_OK;
}

int KvPages::reserve(int seq, int pos, int n, std::vector<int> &src, std::vector<int> &dst)
{
    if (!seq_ok(seq) || pos < 0 || n < 0 || (long long)pos + n > (long long)max_pages_ * KV_PAGE) return E_ARG;
    if (n == 0) return E_OK;
    if (need(seq, pos, n) > free_count()) return E_NOMEM;
    int *t = row(seq);
    for (int i = pos / KV_PAGE; i <= (pos + n - 1) / KV_PAGE; i++) {
        if (t[i] >= 0 && refs_[t[i]] == 1) continue;
        const int p = take();
        if (t[i] >= 0) {
            src.push_back(t[i]);
            dst.push_back(p);
            drop(t[i]);
        }
        t[i] = p;
    }
    return E_OK;
}

int KvPages::fork(int src, int dst, int len)
{
    if (!seq_ok(src) || !seq_ok(dst) || src == dst || len < 0 || len > len_[src]) return E_ARG;
    truncate(dst, 0);
    const int *s = row(src);
    int *d = row(dst);
    for (int i = 0; i < (len + KV_PAGE - 1) / KV_PAGE; i++) {
        d[i] = s[i];
        refs_[s[i]]++;
    }
    len_[dst] = len;
    return E_OK;
}

int KvPages::truncate(int seq, int len)
{
    if (!seq_ok(seq) || len < 0 || len > len_[seq]) return E_ARG;
    int *t = row(seq);
    for (int i = (len + KV_PAGE - 1) / KV_PAGE; i < max_pages_ && t[i] >= 0; i++) {
        drop(t[i]);
        t[i] = -1;
    }
    len_[seq] = len;
    return E_OK;
}

void KvPages::compact(std::vector<int> &src, std::vector<int> &dst)
{
    const int used = n_pages() - free_count();
    std::vector<int> to(n_pages(), -1);
    auto hole = free_.begin();
    for (int p = used; p < n_pages(); p++) {
        if (!refs_[p]) continue;
        to[p] = *hole++;   // as many holes below `used` as used pages from it on
        src.push_back(p);
        dst.push_back(to[p]);
    }
    if (src.empty()) return;
    for (size_t i = 0; i < src.size(); i++) {
        refs_[dst[i]] = refs_[src[i]];
        refs_[src[i]] = 0;
    }
    for (int &p : table_)
        if (p >= 0 && to[p] >= 0) p = to[p];
    free_.clear();
    for (int p = used; p < n_pages(); p++) free_.insert(free_.end(), p);
}

} // namespace cats

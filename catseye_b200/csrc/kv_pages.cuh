// kv_pages.cuh — which page of a paged cache holds which tokens of which
// sequence: host bookkeeping only, the pages' contents are kv.cu's.
#pragma once
#include "kv.cuh"
#include <set>
#include <vector>

namespace cats {

// A page may stand in several sequences' tables (a fork); it is copied when
// one of them writes into it.  The lowest free page is taken first.
class KvPages {
public:
    KvPages(int n_pages, int n_seqs, int max_pages);

    // Make positions pos .. pos + n - 1 of a sequence writable: pages it lacks
    // are taken, pages it shares are replaced (the copies to make are appended
    // to src / dst).  pos may not lie past the sequence's end (E_ARG: the gap
    // would be read).  E_NOMEM, with nothing changed, when too few are free.
    int write(int seq, int pos, int n, std::vector<int> &src, std::vector<int> &dst);
    // The same without the tokens being there yet: the length stays until count()
    // says that a sequence holds its first `end` tokens.  (pos may lie behind
    // other reserved positions.)  truncate() frees what was reserved and not
    // counted.
    int reserve(int seq, int pos, int n, std::vector<int> &src, std::vector<int> &dst);
    void count(int seq, int end) { if (end > len_[seq]) len_[seq] = end; }
    // dst becomes the first len tokens of src, sharing its pages.
    int fork(int src, int dst, int len);
    // Keep the first len tokens of a sequence, and pages for no more; pages nobody holds are free.
    int truncate(int seq, int len);
    // Renumber so that the used pages are 0 .. used - 1 (the copies to make).
    void compact(std::vector<int> &src, std::vector<int> &dst);

    int need(int seq, int pos, int n) const;   // pages that write() would take
    int length(int seq) const { return len_[seq]; }
    int free_count() const { return (int)free_.size(); }
    int n_pages() const { return (int)refs_.size(); }
    int n_seqs() const { return (int)len_.size(); }
    int max_pages() const { return max_pages_; }
    const int *table() const { return table_.data(); }
    bool seq_ok(int s) const { return s >= 0 && s < n_seqs(); }

private:
    int *row(int seq) { return table_.data() + (size_t)seq * max_pages_; }
    const int *row(int seq) const { return table_.data() + (size_t)seq * max_pages_; }
    int take();
    void drop(int page);

    int max_pages_;
    std::vector<int> table_, refs_, len_;
    std::set<int> free_;
};

} // namespace cats

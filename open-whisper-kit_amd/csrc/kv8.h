// The 8-bit key/value cache (include/owk_kv8.h): what its kernels (k_kv8.hip) take once the C entries
// (kv8.cpp) have checked a call.
#pragma once

#include "common.h"
#include "owk_kv8.h"

namespace owk {

struct Kv8Rows {
    char * p = nullptr;
    int64_t entry = 0, row = 0, head = 0;  // element strides
    bool vec = false;                      // every head of every row starts on a 16-byte boundary
};

struct Kv8Call {
    owk_kv8_cache c;
    owk_kv8_batch b;
};

constexpr int kKv8Block = OWK_KV8_BLOCK;

template <typename I> __host__ __device__ inline I kv8_min(I a, I b) { return a < b ? a : b; }
template <typename I> __host__ __device__ inline I kv8_max(I a, I b) { return a > b ? a : b; }

// one entry of a call, bounded by what the cache and the tensors hold: what a caller can get wrong on the
// device (a sequence, a length, an offset, a table entry) leads to nothing here, never out of a tensor
struct Kv8Entry {
    int seq;       // -1: no such sequence
    int start;     // tokens held before the call's own
    int n;         // the call's own tokens / rows
    int64_t row0;  // first row in a joined tensor; in a padded one 0 (its entry stride leads there)
};

__host__ __device__ inline Kv8Entry kv8_entry(const Kv8Call & a, int b) {
    Kv8Entry e;
    const int cap = a.c.max_blocks * kKv8Block;
    e.seq = a.b.seq ? a.b.seq[b] : b;
    if (e.seq < 0 || e.seq >= a.c.n_seqs) e.seq = -1;
    e.start = kv8_min(kv8_max(a.b.lens[b], 0), cap);
    e.row0 = 0;
    if (a.b.off) {
        const int64_t lo = a.b.off[b], hi = kv8_min((int64_t) a.b.off[b + 1], a.b.rows);
        e.row0 = lo;
        e.n = lo < 0 || hi <= lo ? 0 : (int) kv8_min(hi - lo, (int64_t) a.b.max_new);
    } else {
        e.n = a.b.count ? kv8_min(kv8_max(a.b.count[b], 0), a.b.max_new) : a.b.max_new;
    }
    return e;
}

// the pool's block that holds block i of a sequence, or -1
__host__ __device__ inline int64_t kv8_page(const owk_kv8_cache & c, int seq, int i) {
    if (seq < 0 || i < 0 || i >= c.max_blocks) return -1;
    const int64_t at = (int64_t) seq * c.max_blocks + i;
    const int64_t p = c.table ? c.table[at] : at;
    return p < 0 || p >= c.n_blocks ? -1 : p;
}

struct Kv8Attend {
    Kv8Rows q, out;
    int group = 1;      // query heads of a key/value head
    int causal = 0;
    int splits = 1;     // parts of `per` blocks that the keys of an entry are cut into at most, a workgroup each
    int per = 0;
    int tiles = 1;      // of 16 rows of an entry and head
    int join = 1;       // of them in a workgroup
    float scale = 1.0f;
    float * ws = nullptr;
};

// the split and workspace of an attend call (host arithmetic on the call's sizes alone)
struct Kv8Plan {
    int splits = 1, per = 0, tiles = 0;
    int join = 1;              // tiles of 16 rows in a workgroup
    bool many = false, wide = false;
    bool fits = true;          // false: more rows or workgroups than a launch can have
    size_t ws_bytes = 0;
};
void kv8_set_many_rows(int rows);  // for tests, of this thread: calls of more rows a head run in many-row tiles; 0: by kv8_plan's own rule
Kv8Plan kv8_plan(const Kv8Call & call, int group, int max_len);

void kv8_append(hipStream_t s, const Kv8Call & call, const Kv8Rows & k, const Kv8Rows & v);
void kv8_attend(hipStream_t s, const Kv8Call & call, const Kv8Attend & a, const Kv8Plan & plan, int out_type);
void kv8_read(hipStream_t s, const Kv8Call & call, const int32_t * first, const Kv8Rows & k, const Kv8Rows & v);

} // namespace owk

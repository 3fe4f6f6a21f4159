// vs_kv.h -- the paged key-value cache's handle, shared by the sources of its
// entry points (vs_attend.hip, vs_pages.hip).
#pragma once

#include "vs_host.h"
#include "vs_internal.h"

struct vs_kv {
    int device = 0;
    int64_t npages = 0, page_size = 0, layers = 0, kv_heads = 0, head_dim = 0;
    int dtype = VS_DTYPE_BF16;
    int64_t page_bytes = 0;
    char *mem = nullptr;
    bool owns_mem = false;
    int num_cu = 256;
    int32_t *status = nullptr;  // kStatusWords device words
    uint8_t *closed = nullptr;  // [npages], behind them: pages that take no new token
    vs::StreamScratch scratch;
};

namespace vs {

// What kernels tell vs_kv_check: [0] bits below, [1] pages an extend was short
// of, [2] whether a page may be closed.
//
// An extend that does not fit is known on the device only, with the calls that
// store what it should have made room for behind it: they would store at the
// last positions that there are, over tokens that are in use, and in pages whose
// copies were part of the refused plan several at once.  So it closes the last
// page of each of its sequences, and those calls leave a sequence alone whose
// last page is closed.  The page is what is marked, not the sequence: that
// follows forks and compactions, and concerns no one else's sequences.  An
// extend that fits opens the pages that it gives or leaves to a sequence,
// vs_kv_check opens all.
constexpr int kStatusWords = 4;
constexpr int kStatusPages = 1, kStatusWidth = 2, kStatusParent = 4, kStatusNoPage = 8;

// Positions per block, the unit of the cache's layout: what one bf16 matrix
// instruction sums over.
constexpr int kKvBlock = 32;

inline int64_t kv_elem(int dtype) { return dtype == VS_DTYPE_BF16 ? 2 : 4; }

inline int check_seqs(const vs_kv *kv, const vs_kv_seqs *s) {
    if (!s) return report(VS_ERR_INVALID, "null sequences");
    if (s->nseq < 0 || s->width < 0)
        return report(VS_ERR_INVALID, "negative number of sequences or table columns");
    if (s->nseq > (1 << 20)) return report(VS_ERR_UNSUPPORTED, "more than 2^20 sequences");
    if (s->width > INT32_MAX / kv->page_size)
        return report(VS_ERR_UNSUPPORTED, "table columns past 2^31 positions");
    if (!s->refs || (s->nseq > 0 && (!s->lens || (!s->table && s->width > 0))))
        return report(VS_ERR_INVALID, "null table, lens or refs");
    if (((uintptr_t)s->table | (uintptr_t)s->lens | (uintptr_t)s->refs) % 4)
        return report(VS_ERR_INVALID, "table, lens or refs are not aligned to their elements");
    return VS_OK;
}

}  // namespace vs

// vs_pages.hip -- the pages of the key-value cache: extending (with copies on
// write), forking, freeing, evicting, compacting and copying.  The tables,
// lengths and reference counts live on the device, so a decoding loop never
// waits for the host to manage them.
#include "vs_kv.h"
#include "vs_wave.h"

namespace vs {
namespace {

constexpr int kSmallPages = 16384;    // of a cache whose compaction is planned in registers
constexpr int kForkSeqs = 1024;      // sequences and words of a fork that one workgroup does
constexpr int kForkWords = 6 << 10;
constexpr int kPieceBytes = 8192;   // of a page, per workgroup pass of the copy

struct ExtendArgs {
    int32_t *table, *lens, *refs;
    int64_t width;
    int nseq, npages, page_shift, count;
    const int32_t *count_dev;
    int32_t *status;
    uint8_t *closed;
    int32_t *holders, *lowest;  // [npages], used where a shared last page is
    int32_t *offset;            // [nseq] place of a sequence's first new page | copies (bit 31)
    int32_t *fresh;             // [npages] free pages, lowest first
    int32_t *copies;            // [0] how many, then pairs (from, to)
};

// Divides the free pages among the sequences, as one workgroup: the work is a
// few thousand numbers, and its steps need each other's results.  What bounds
// it is the chain of loads (length, table entry, count), so a thread keeps what
// it reads of its first sequence, the first pages' counts are read beside it,
// and up to kPlan sequences meet on their shared pages in LDS (SMALL).  4
// sequences 4.0 us, 256 of them 5.7 (with tables in memory 9).
template <bool SMALL>
__global__ __launch_bounds__(kPlan) void extend_plan_kernel(ExtendArgs a) {
    constexpr int kHash = 2 * kPlan;
    __shared__ int lds[kPlan / 64];
    __shared__ int bad;
    __shared__ int h_page[SMALL ? kHash : 1], h_holders[SMALL ? kHash : 1], h_lowest[SMALL ? kHash : 1];
    __shared__ int fresh[4 * kPlan];  // the first free pages that are needed
    const int P = 1 << a.page_shift;
    const int64_t most = a.width << a.page_shift;
    int refs0[4];  // of the first 4 kPlan pages
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t p = 4 * threadIdx.x + i;
        refs0[i] = p < a.npages ? a.refs[p] : 1;
    }
    struct Seq {
        int n, count, page, refs;  // page: a partly filled last page that others hold too, or -1
    };
    auto read = [&](int b) {
        Seq s = {0, 0, -1, 0};
        if (b >= a.nseq) return s;
        s.n = max(a.lens[b], 0);
        s.count = max(a.count_dev ? a.count_dev[b] : a.count, 0);
        if ((s.n & (P - 1)) && s.n <= most && s.count) {
            const int p = a.table[(int64_t)b * a.width + ((s.n - 1) >> a.page_shift)];
            if ((unsigned)p < (unsigned)a.npages) {
                s.refs = a.refs[p];
                if (s.refs > 1) s.page = p;
            }
        }
        return s;
    };
    const bool marked = a.status[2] != 0;  // some page may be closed
    if (threadIdx.x == 0) {
        bad = 0;
        a.copies[0] = 0;
    }
    if constexpr (SMALL) {
        for (int i = threadIdx.x; i < kHash; i += kPlan) {
            h_page[i] = -1;
            h_holders[i] = 0;
            h_lowest[i] = INT32_MAX;
        }
    }
    const Seq first = read(threadIdx.x);
    int place = 0;  // of its page in the hash table
    __syncthreads();
    if constexpr (SMALL) {
        if (first.page >= 0) {
            place = (int)((uint32_t)first.page * 2654435761u >> 21) & (kHash - 1);
            for (;;) {  // (at most kPlan pages in 2 kPlan places: one is free)
                const int was = atomicCAS(&h_page[place], -1, first.page);
                if (was == -1 || was == first.page) break;
                place = (place + 1) & (kHash - 1);
            }
            atomicAdd(&h_holders[place], 1);
            atomicMin(&h_lowest[place], (int)threadIdx.x);
        }
    } else {
        for (int b = threadIdx.x; b < a.nseq; b += kPlan) {
            const int p = read(b).page;
            if (p >= 0) {
                a.holders[p] = 0;
                a.lowest[p] = INT32_MAX;
            }
        }
        __syncthreads();
        for (int b = threadIdx.x; b < a.nseq; b += kPlan) {
            const int p = read(b).page;
            if (p >= 0) {
                atomicAdd(&a.holders[p], 1);
                atomicMin(&a.lowest[p], b);
            }
        }
    }
    __syncthreads();
    int64_t need = 0;  // (equal in all threads)
    int at0 = 0;       // the thread's first sequence's first new page; its copy
    bool copy0 = false;
    for (int b0 = 0; b0 < a.nseq; b0 += kPlan) {
        const int b = b0 + threadIdx.x;
        const Seq s = b0 ? read(b) : first;
        int want = 0;
        bool copy = false;
        if (s.count && (int64_t)s.n + s.count > most) {
            bad = 1;
        } else if (s.count) {
            if (s.page >= 0) {
                if constexpr (SMALL)
                    copy = !(h_lowest[place] == b && h_holders[place] == s.refs);
                else
                    copy = !(a.lowest[s.page] == b && a.holders[s.page] == s.refs);
            }
            want = copy + (int)(((int64_t)s.n + s.count + P - 1) >> a.page_shift) -
                   (int)(((int64_t)s.n + P - 1) >> a.page_shift);
        }
        // (a total that 32 bits cannot hold is more than there are pages: refused)
        uint32_t total;
        const int at = (int)min(need + block_scan_sat((uint32_t)want, &total, lds), (int64_t)INT32_MAX);
        if (b0 == 0) {
            at0 = at;
            copy0 = copy;
        }
        if (!SMALL && b < a.nseq) a.offset[b] = at | (copy ? (int)0x80000000 : 0);
        need += total;
    }
    __syncthreads();
    // what is stored behind a refused extend has no place: see kStatusWords
    auto close_pages = [&]() {
        for (int b = threadIdx.x; b < a.nseq; b += kPlan) {
            const int n = max(a.lens[b], 0);
            if (n == 0 || n > most || (a.count_dev ? a.count_dev[b] : a.count) <= 0) continue;
            const int p = a.table[(int64_t)b * a.width + ((n - 1) >> a.page_shift)];
            if ((unsigned)p < (unsigned)a.npages) a.closed[p] = 1;
        }
        if (threadIdx.x == 0) a.status[2] = 1;
    };
    if (bad) {
        if (threadIdx.x == 0) atomicOr(&a.status[0], kStatusWidth);
        close_pages();
        return;
    }
    // the lowest `need` free pages, the first in LDS
    int64_t found = 0;
    for (int64_t p0 = 0; p0 < a.npages && found < need; p0 += 4 * kPlan) {
        int free[4], cnt = 0;
        const int64_t p = p0 + 4 * threadIdx.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            free[i] = p0 ? p + i < a.npages && a.refs[p + i] == 0 : refs0[i] == 0;
            cnt += free[i];
        }
        int total, at = block_scan(cnt, &total, lds);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (free[i]) {
                const int64_t x = found + at++;
                if (x >= need) continue;
                if (x < 4 * kPlan)
                    fresh[x] = (int)(p + i);
                else
                    a.fresh[x] = (int)(p + i);
            }
        found += total;
    }
    if (found < need) {
        if (threadIdx.x == 0) {
            atomicOr(&a.status[0], kStatusPages);
            atomicMax(&a.status[1], (int)min(max(need - found, (int64_t)1), (int64_t)INT32_MAX));
        }
        close_pages();
        return;
    }
    __syncthreads();
    auto take = [&](int x) { return x < 4 * kPlan ? fresh[x] : a.fresh[x]; };
    for (int b = threadIdx.x; b < a.nseq; b += kPlan) {
        const bool mine = b == (int)threadIdx.x;
        const int n = mine ? first.n : max(a.lens[b], 0);
        const int c = mine ? first.count : max(a.count_dev ? a.count_dev[b] : a.count, 0);
        if (!c) continue;
        int at = mine ? at0 : a.offset[b] & 0x7FFFFFFF;
        int32_t *row = a.table + (int64_t)b * a.width;
        if (mine ? copy0 : a.offset[b] < 0) {
            int32_t *entry = &row[(n - 1) >> a.page_shift];
            const int from = mine ? first.page : *entry, to = take(at++);
            const int i = atomicAdd(&a.copies[0], 1);  // (their order does not matter)
            a.copies[1 + 2 * i] = from;
            a.copies[2 + 2 * i] = to;
            atomicSub(&a.refs[from], 1);
            a.refs[to] = 1;
            *entry = to;
        }
        if (marked && (n & (P - 1))) {  // (a full one may be others' last page too)
            const int p = row[(n - 1) >> a.page_shift];
            if ((unsigned)p < (unsigned)a.npages) a.closed[p] = 0;
        }
        const int64_t end = ((int64_t)n + c + P - 1) >> a.page_shift;
        for (int64_t e = ((int64_t)n + P - 1) >> a.page_shift; e < end; ++e) {
            const int to = take(at++);
            a.refs[to] = 1;
            row[e] = to;
            if (marked) a.closed[to] = 0;
        }
        a.lens[b] = n + c;
    }
}

// Copies pages: HBM-bound.  Nothing is read twice, so loads and stores pass the
// caches by, and many small pieces spread best (1.03 GB of pages: 417 us with
// cached accesses, 401 without, 390 in 8 KB pieces by 32 workgroups to a CU:
// 5.3 TB/s read and written; 370 to 380 by card).  The grid walks (page, piece) pairs; `n_dev` is
// read on the device because the host does not know how many pages a plan moves.
// Compaction's tables (`tables`) are rewritten on the way.
struct Tables {
    const int32_t *table, *lens, *map;
    int32_t *table2, *lens2;
    int64_t entries;
    int nseq;
};

__global__ __launch_bounds__(256) void copy_pages_kernel(char *pool, int64_t page_bytes, int npages,
                                                         const int32_t *n_dev, int64_t n_host,
                                                         const int32_t *from, const int32_t *to,
                                                         int stride, Tables tables) {
    const int64_t every = (int64_t)gridDim.x * 256;
    for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < tables.entries; x += every) {
        const int p = tables.table[x];
        tables.table2[x] = (unsigned)p < (unsigned)npages ? tables.map[p] : p;
    }
    for (int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x; b < tables.nseq; b += every)
        tables.lens2[b] = tables.lens[b];
    const int64_t n = n_dev ? *n_dev : n_host;
    const int64_t pieces = (page_bytes + kPieceBytes - 1) / kPieceBytes;
    for (int64_t w = blockIdx.x; w < n * pieces; w += gridDim.x) {
        const int64_t i = w / pieces, x0 = w % pieces * kPieceBytes;
        const int f = from[i * stride], t = to[i * stride];
        if ((unsigned)f >= (unsigned)npages || (unsigned)t >= (unsigned)npages) continue;
        const char *src = pool + f * page_bytes + x0;
        char *dst = pool + t * page_bytes + x0;
        const int bytes = (int)min((int64_t)kPieceBytes, page_bytes - x0);
        u32x4_t v[kPieceBytes / 4096];
#pragma unroll
        for (int k = 0; k < kPieceBytes / 4096; ++k) {
            const int x = k * 4096 + threadIdx.x * 16;
            if (x < bytes) v[k] = __builtin_nontemporal_load((const u32x4_t *)(src + x));
        }
#pragma unroll
        for (int k = 0; k < kPieceBytes / 4096; ++k) {
            const int x = k * 4096 + threadIdx.x * 16;
            if (x < bytes) __builtin_nontemporal_store(v[k], (u32x4_t *)(dst + x));
        }
    }
}

// Another table whose pages compaction moved: two loads and a store per entry.
__global__ __launch_bounds__(256) void remap_kernel(int32_t *table, int64_t entries, int npages,
                                                    const int32_t *map) {
    for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < entries;
         x += (int64_t)gridDim.x * 256) {
        const int p = table[x];
        if ((unsigned)p < (unsigned)npages) table[x] = map[p];
    }
}

struct ForkArgs {
    const int32_t *table, *lens, *parents;
    int32_t *table2, *lens2, *refs;
    int64_t width;
    int nin, nout, npages;
    int32_t *status;
};

__global__ __launch_bounds__(256) void copy_words_kernel(const int32_t *in, int32_t *out, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
        out[i] = in[i];
}

// One workgroup per sequence of either side: two loads and an atomic per table
// entry, so latency is what it takes (256 sequences of 36 entries 2.8 to 4 us,
// and the copy of the counts before it as long again).  References are whole numbers,
// so the order of the atomics changes nothing.
__global__ __launch_bounds__(256) void fork_kernel(ForkArgs a) {
    __shared__ int part[4];
    for (int w = blockIdx.x; w < a.nin + a.nout; w += gridDim.x) {
        if (w < a.nout) {
            int parent = a.parents[w];
            const bool ok = (unsigned)parent < (unsigned)a.nin;
            if (!ok && parent != -1 && threadIdx.x == 0) atomicOr(&a.status[0], kStatusParent);
            for (int64_t x = threadIdx.x; x < a.width; x += 256)
                a.table2[w * a.width + x] = ok ? a.table[parent * a.width + x] : -1;
            if (threadIdx.x == 0) a.lens2[w] = ok ? a.lens[parent] : 0;
        } else {
            const int b = w - a.nout;
            int c = 0;
            for (int i = threadIdx.x; i < a.nout; i += 256) c += a.parents[i] == b;
#pragma unroll
            for (int d = 32; d; d >>= 1) c += __shfl_xor(c, d);
            __syncthreads();
            if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = c;
            __syncthreads();
            c = part[0] + part[1] + part[2] + part[3] - 1;
            if (c)
                for (int64_t x = threadIdx.x; x < a.width; x += 256) {
                    const int p = a.table[b * a.width + x];
                    if ((unsigned)p < (unsigned)a.npages) atomicAdd(&a.refs[p], c);
                }
        }
    }
}

// The same as one workgroup, where that takes less than a second launch: the
// counts are copied, then changed.  By the words that it goes through (pages,
// and table entries and lengths of both sides), one workgroup against two launches:
// 216 (96 pages, 4 sequences of 14 entries) 2.4 and 3.5 us, 1,672 (1,000, 16 of
// 20) 2.4 and 3.8, 2,920 (1,000, 64 of 14) 2.8 and 3.9, 4,968 (1,000, 64 of 30) 3.6
// and 3.8, 5,840 (2,000, 128 of 14) 3.5 and 3.9, 6,248 (6,000, 4 of 30) 3.1 and 3.6;
// 8,936 (1,000, 128 of 30) 4.7 and 3.8, 10,624 (8,000, 32 of 40) 4.1 and 3.9, 22,444
// (3,500, 256 of 36) 8.8 and 4.0.  Hence kForkWords.
__global__ __launch_bounds__(kPlan) void fork_small_kernel(ForkArgs a, const int32_t *refs_in) {
    __shared__ int children[kForkSeqs], parent_of[kForkSeqs];
    for (int i = threadIdx.x; i < a.nin; i += kPlan) children[i] = 0;
    if (refs_in != a.refs) {
#pragma unroll 4
        for (int i = threadIdx.x; i < a.npages; i += kPlan) a.refs[i] = refs_in[i];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.nout; i += kPlan) {
        int parent = a.parents[i];
        if ((unsigned)parent < (unsigned)a.nin) {
            atomicAdd(&children[parent], 1);
        } else {
            if (parent != -1) atomicOr(&a.status[0], kStatusParent);
            parent = -1;
        }
        parent_of[i] = parent;
        a.lens2[i] = parent >= 0 ? a.lens[parent] : 0;
    }
    __syncthreads();
    const uint32_t width = (uint32_t)a.width, entries = (uint32_t)a.nin * width;
#pragma unroll 4
    for (uint32_t x = threadIdx.x; x < (uint32_t)a.nout * width; x += kPlan) {
        const int parent = parent_of[x / width];
        a.table2[x] = parent >= 0 ? a.table[(uint32_t)parent * width + x % width] : -1;
    }
#pragma unroll 4
    for (uint32_t x = threadIdx.x; x < entries; x += kPlan) {
        const int c = children[x / width] - 1, p = a.table[x];
        if (c && (unsigned)p < (unsigned)a.npages) atomicAdd(&a.refs[p], c);
    }
}

// A few atomics per thread: 1.4 us for a sequence, 2.4 for 16 of 32 entries.
__global__ __launch_bounds__(256) void free_kernel(int32_t *table, int32_t *lens, int32_t *refs,
                                                   int64_t width, int nseq, int npages,
                                                   const int32_t *ids, int64_t n) {
    for (int64_t w = blockIdx.x; w < n; w += gridDim.x) {
        const int b = ids ? ids[w] : (int)w;
        if ((unsigned)b >= (unsigned)nseq) continue;
        for (int64_t x = threadIdx.x; x < width; x += 256) {
            // (whoever takes the entry gives its reference back: once)
            const int p = atomicExch(&table[b * width + x], -1);
            if ((unsigned)p < (unsigned)npages) atomicSub(&refs[p], 1);
        }
        if (threadIdx.x == 0) lens[b] = 0;
    }
}

// The same for a sequence's pages behind the window, 1.3 to 2.4 us.
__global__ __launch_bounds__(256) void evict_kernel(int32_t *table, const int32_t *lens,
                                                    int32_t *refs, int64_t width, int nseq,
                                                    int npages, int page_shift, int64_t window,
                                                    int64_t sinks) {
    for (int b = blockIdx.x; b < nseq; b += gridDim.x) {
        // pages [lo, hi) hold no visible position, now or later
        const int64_t size = (int64_t)1 << page_shift;
        const int64_t lo = (min(sinks, (int64_t)1 << 31) + size - 1) >> page_shift;
        const int64_t hi = min((lens[b] - window) >> page_shift, width);
        for (int64_t x = lo + threadIdx.x; x < hi; x += 256) {
            const int p = table[b * width + x];
            if ((unsigned)p < (unsigned)npages) {
                atomicSub(&refs[p], 1);
                table[b * width + x] = -1;
            }
        }
    }
}

struct CompactArgs {
    const int32_t *refs;
    int32_t *refs2;
    int npages;
    int32_t *map;      // [npages] where a page goes
    int32_t *from, *to;
    int32_t *moves;    // how many
    const int32_t *status;
    uint8_t *closed;   // follows its pages
};

// Live pages past the front and free pages in it, paired in order.  Bound by one
// workgroup's passes over the counts, small beside the pages' copy.
__global__ __launch_bounds__(kPlan) void compact_plan_kernel(CompactArgs a) {
    __shared__ int lds[kPlan / 64];
    const int64_t step = 4 * kPlan;
    const bool marked = a.status[2] != 0;
    int64_t live = 0;
    for (int64_t p0 = 0; p0 < a.npages; p0 += step) {
        int cnt = 0;
        const int64_t p = p0 + 4 * threadIdx.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) cnt += p + i < a.npages && a.refs[p + i] != 0;
        int total;
        block_scan(cnt, &total, lds);
        live += total;
    }
    int nto = 0, nfrom = 0;
    for (int64_t p0 = 0; p0 < a.npages; p0 += step) {
        int ref[4], cnt = 0;
        const int64_t p = p0 + 4 * threadIdx.x;
        // free pages of the front count 1, live pages past it 2^16: both are at most 4096 here
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            ref[i] = p + i < a.npages ? a.refs[p + i] : 0;
            if (p + i >= a.npages) continue;
            if (p + i < live)
                cnt += ref[i] == 0;
            else
                cnt += (ref[i] != 0) << 16;
        }
        int total;
        const int at = block_scan(cnt, &total, lds);
        int t = nto + (at & 0xFFFF), f = nfrom + (at >> 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (p + i >= a.npages) continue;
            a.map[p + i] = (int)(p + i);
            if (p + i < live) {
                a.refs2[p + i] = ref[i];
                if (ref[i] == 0) a.to[t++] = (int)(p + i);
            } else {
                if (ref[i] != 0) a.from[f++] = (int)(p + i);
            }
        }
        nto += total & 0xFFFF;
        nfrom += total >> 16;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < nto; i += kPlan) {
        const int f = a.from[i], t = a.to[i];
        a.map[f] = t;
        a.refs2[t] = a.refs[f];
        if (marked) {
            a.closed[t] = a.closed[f];
            a.closed[f] = 0;
        }
    }
    __syncthreads();
    for (int64_t p = live + threadIdx.x; p < a.npages; p += kPlan) a.refs2[p] = 0;
    if (threadIdx.x == 0) *a.moves = nto;
}

// The same for up to kSmallPages pages: the counts are read once, into
// registers, and the pairs meet in LDS (150 pages 3.2 us, 4,100 pages 7.0).
__global__ __launch_bounds__(kPlan) void compact_plan_small_kernel(CompactArgs a) {
    constexpr int N = kSmallPages / (4 * kPlan);  // rounds of four consecutive pages per thread
    __shared__ int lds[kPlan / 64];
    __shared__ uint16_t to[kSmallPages / 2];
    const int chunks = (a.npages + 4 * kPlan - 1) / (4 * kPlan);
    const bool marked = a.status[2] != 0;
    int ref[N][4], cnt = 0;
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = (c * kPlan + threadIdx.x) * 4 + i;
            ref[c][i] = p < a.npages ? a.refs[p] : 0;
            cnt += ref[c][i] != 0;
        }
    int live, total, done = 0, at[N];
    block_scan(cnt, &live, lds);
    // free pages of the front count 1, live pages past it 2^16
#pragma unroll
    for (int c = 0; c < N; ++c) {
        if (c >= chunks) break;
        cnt = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = (c * kPlan + threadIdx.x) * 4 + i;
            if (p < a.npages) cnt += p < live ? ref[c][i] == 0 : (ref[c][i] != 0) << 16;
        }
        at[c] = done + block_scan(cnt, &total, lds);
        done += total;
        int t = at[c] & 0xFFFF;  // the thread's place in the list of free pages
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = (c * kPlan + threadIdx.x) * 4 + i;
            if (p >= a.npages) continue;
            if (p < live && ref[c][i] == 0) to[t++] = (uint16_t)p;
            a.refs2[p] = p < live ? ref[c][i] : 0;
            a.map[p] = p;
        }
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < N; ++c) {
        if (c >= chunks) break;
        int f = at[c] >> 16;  // and in that of pages to move
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = (c * kPlan + threadIdx.x) * 4 + i;
            if (p >= a.npages || p < live || ref[c][i] == 0) continue;
            const int dst = to[f];
            a.map[p] = dst;
            a.refs2[dst] = ref[c][i];
            a.from[f] = p;
            a.to[f] = dst;
            if (marked) {
                a.closed[dst] = a.closed[p];
                a.closed[p] = 0;
            }
            ++f;
        }
    }
    if (threadIdx.x == 0) *a.moves = done & 0xFFFF;
}

hipError_t launch_copy(const vs_kv *kv, const int32_t *n_dev, int64_t n_max, const int32_t *from,
                       const int32_t *to, int stride, hipStream_t st, const Tables &tables = {}) {
    const int64_t pieces = (kv->page_bytes + kPieceBytes - 1) / kPieceBytes;
    const int64_t wgs = std::min<int64_t>((int64_t)kv->num_cu * 32,
                                          std::max(n_max * pieces, (tables.entries + 255) / 256));
    if (wgs <= 0) return hipSuccess;
    hipLaunchKernelGGL(copy_pages_kernel, dim3((uint32_t)wgs), dim3(256), 0, st, kv->mem,
                       kv->page_bytes, (int)kv->npages, n_dev, n_max, from, to, stride, tables);
    return hipGetLastError();
}

uint32_t grid_of(int64_t n, int64_t most) { return (uint32_t)std::max<int64_t>(1, std::min(n, most)); }

}  // namespace
}  // namespace vs

using vs::report;
using vs::report_hip;

#define VS_LAUNCHED(what)                                   \
    do {                                                    \
        hipError_t e_ = hipGetLastError();                  \
        if (e_ != hipSuccess) return report_hip(e_, what);  \
    } while (0)

extern "C" {

int vs_kv_extend(vs_kv *kv, const vs_kv_seqs *s, int64_t count, const int32_t *count_dev,
                 void *stream) {
    if (!kv) return report(VS_ERR_INVALID, "null handle");
    int rc = vs::check_seqs(kv, s);
    if (rc) return rc;
    if (!count_dev && (count < 0 || count > INT32_MAX))
        return report(VS_ERR_INVALID, "count %lld", (long long)count);
    if ((uintptr_t)count_dev % 4) return report(VS_ERR_INVALID, "counts are not aligned");
    if (s->nseq == 0 || (!count_dev && count == 0)) return VS_OK;
    vs::DeviceGuard g(kv->device);
    if (g.err != hipSuccess) return report_hip(g.err, "hipSetDevice");
    hipStream_t st = (hipStream_t)stream;
    const int64_t np = kv->npages, ns = s->nseq;
    void *ws = nullptr;
    rc = kv->scratch.get(st, (size_t)(3 * np + 3 * ns + 1) * sizeof(int32_t), &ws);
    if (rc) return rc;
    vs::ExtendArgs a = {};
    a.table = s->table;
    a.lens = s->lens;
    a.refs = s->refs;
    a.width = s->width;
    a.nseq = (int)ns;
    a.npages = (int)np;
    a.page_shift = __builtin_ctzll((uint64_t)kv->page_size);
    a.count = (int)count;
    a.count_dev = count_dev;
    a.status = kv->status;
    a.closed = kv->closed;
    a.holders = (int32_t *)ws;
    a.lowest = a.holders + np;
    a.fresh = a.lowest + np;
    a.offset = a.fresh + np;
    a.copies = a.offset + ns;
    if (ns <= vs::kPlan)
        hipLaunchKernelGGL(vs::extend_plan_kernel<true>, dim3(1), dim3(vs::kPlan), 0, st, a);
    else
        hipLaunchKernelGGL(vs::extend_plan_kernel<false>, dim3(1), dim3(vs::kPlan), 0, st, a);
    VS_LAUNCHED("extend");
    hipError_t e = vs::launch_copy(kv, a.copies, ns, a.copies + 1, a.copies + 2, 2, st);
    return e == hipSuccess ? VS_OK : report_hip(e, "page copies");
}

int vs_kv_fork(vs_kv *kv, const vs_kv_seqs *in, const int32_t *parents, const vs_kv_seqs *out,
               void *stream) {
    if (!kv) return report(VS_ERR_INVALID, "null handle");
    int rc = vs::check_seqs(kv, in);
    if (!rc) rc = vs::check_seqs(kv, out);
    if (rc) return rc;
    if (in->width != out->width)
        return report(VS_ERR_INVALID, "tables of %lld and %lld columns", (long long)in->width,
                      (long long)out->width);
    const int64_t in_table = in->nseq * in->width * 4, out_table = out->nseq * out->width * 4;
    if ((in->nseq && in->lens == out->lens) || (in->table == out->table && in->width) ||
        vs::overlap(in->lens, in->nseq * 4, out->lens, out->nseq * 4) ||
        vs::overlap(in->table, in_table, out->table, out_table))
        return report(VS_ERR_INVALID, "fork needs another table and other lens to write to");
    if ((out->nseq && !parents) || (uintptr_t)parents % 4)
        return report(VS_ERR_INVALID, "null or unaligned parents");
    if (vs::overlap(parents, out->nseq * 4, out->table, out_table) ||
        vs::overlap(parents, out->nseq * 4, out->lens, out->nseq * 4))
        return report(VS_ERR_INVALID, "fork: parents lie in out");
    if (in->refs != out->refs &&
        vs::overlap(in->refs, kv->npages * 4, out->refs, kv->npages * 4))
        return report(VS_ERR_INVALID, "fork: counts that overlap in part");
    vs::DeviceGuard g(kv->device);
    if (g.err != hipSuccess) return report_hip(g.err, "hipSetDevice");
    hipStream_t st = (hipStream_t)stream;
    vs::ForkArgs a = {};
    a.table = in->table;
    a.lens = in->lens;
    a.parents = parents;
    a.table2 = out->table;
    a.lens2 = out->lens;
    a.refs = out->refs;
    a.width = in->width;
    a.nin = (int)in->nseq;
    a.nout = (int)out->nseq;
    a.npages = (int)kv->npages;
    a.status = kv->status;
    const int64_t both = in->nseq + out->nseq;
    if (std::max(in->nseq, out->nseq) <= vs::kForkSeqs && kv->npages + both * (in->width + 1) < vs::kForkWords) {
        hipLaunchKernelGGL(vs::fork_small_kernel, dim3(1), dim3(vs::kPlan), 0, st, a, in->refs);
        VS_LAUNCHED("fork");
        return VS_OK;
    }
    if (in->refs != out->refs) {
        hipLaunchKernelGGL(vs::copy_words_kernel, dim3(vs::grid_of((kv->npages + 255) / 256, 2048)),
                           dim3(256), 0, st, in->refs, out->refs, kv->npages);
        VS_LAUNCHED("fork");
    }
    if (both == 0) return VS_OK;
    hipLaunchKernelGGL(vs::fork_kernel, dim3(vs::grid_of(both, 65536)), dim3(256), 0, st, a);
    VS_LAUNCHED("fork");
    return VS_OK;
}

int vs_kv_free(vs_kv *kv, const vs_kv_seqs *s, const int32_t *ids, int64_t n, void *stream) {
    if (!kv) return report(VS_ERR_INVALID, "null handle");
    int rc = vs::check_seqs(kv, s);
    if (rc) return rc;
    if (ids && n < 0) return report(VS_ERR_INVALID, "n %lld", (long long)n);
    if ((uintptr_t)ids % 4) return report(VS_ERR_INVALID, "ids are not aligned");
    if (!ids) n = s->nseq;
    if (n == 0 || s->nseq == 0) return VS_OK;
    vs::DeviceGuard g(kv->device);
    if (g.err != hipSuccess) return report_hip(g.err, "hipSetDevice");
    hipLaunchKernelGGL(vs::free_kernel, dim3(vs::grid_of(n, 65536)), dim3(256), 0,
                       (hipStream_t)stream, s->table, s->lens, s->refs, s->width, (int)s->nseq,
                       (int)kv->npages, ids, n);
    VS_LAUNCHED("free");
    return VS_OK;
}

int vs_kv_evict(vs_kv *kv, const vs_kv_seqs *s, int64_t window, int64_t sinks, void *stream) {
    if (!kv) return report(VS_ERR_INVALID, "null handle");
    int rc = vs::check_seqs(kv, s);
    if (rc) return rc;
    if (window <= 0 || sinks < 0)
        return report(VS_ERR_INVALID, "evict needs a window > 0 and sinks >= 0");
    if (s->nseq == 0 || window > INT32_MAX) return VS_OK;
    vs::DeviceGuard g(kv->device);
    if (g.err != hipSuccess) return report_hip(g.err, "hipSetDevice");
    hipLaunchKernelGGL(vs::evict_kernel, dim3(vs::grid_of(s->nseq, 65536)), dim3(256), 0,
                       (hipStream_t)stream, s->table, s->lens, s->refs, s->width, (int)s->nseq,
                       (int)kv->npages, __builtin_ctzll((uint64_t)kv->page_size), window, sinks);
    VS_LAUNCHED("evict");
    return VS_OK;
}

int vs_kv_compact(vs_kv *kv, const vs_kv_seqs *in, const vs_kv_seqs *out, void *stream) {
    return vs_kv_compact_with(kv, in, out, nullptr, 0, nullptr, stream);
}

int vs_kv_compact_with(vs_kv *kv, const vs_kv_seqs *in, const vs_kv_seqs *out,
                       const vs_kv_seqs *const *others, int64_t nothers, int32_t *map,
                       void *stream) {
    if (!kv) return report(VS_ERR_INVALID, "null handle");
    int rc = vs::check_seqs(kv, in);
    if (!rc) rc = vs::check_seqs(kv, out);
    if (rc) return rc;
    if (in->width != out->width || in->nseq != out->nseq)
        return report(VS_ERR_INVALID, "compact: in and out differ in shape");
    const int64_t table_bytes = in->nseq * in->width * 4;
    if ((in->table != out->table && vs::overlap(in->table, table_bytes, out->table, table_bytes)) ||
        (in->lens != out->lens && vs::overlap(in->lens, in->nseq * 4, out->lens, in->nseq * 4)) ||
        (in->refs != out->refs && vs::overlap(in->refs, kv->npages * 4, out->refs, kv->npages * 4)))
        return report(VS_ERR_INVALID, "compact: in and out overlap in part");
    if (nothers < 0 || (nothers && !others) || (uintptr_t)map % 4)
        return report(VS_ERR_INVALID, "null others, or an unaligned map");
    if (nothers && in->refs != out->refs)
        return report(VS_ERR_INVALID, "others stay on their counts: in and out have to share them");
    for (int64_t i = 0; i < nothers; ++i) {
        rc = vs::check_seqs(kv, others[i]);
        if (rc) return rc;
        if (others[i]->refs != in->refs)
            return report(VS_ERR_INVALID, "other %lld is on other counts", (long long)i);
        // (a table that is rewritten twice would follow its pages twice)
        auto same = [&](const vs_kv_seqs *s) {
            return vs::overlap(others[i]->table, others[i]->nseq * others[i]->width * 4, s->table,
                               s->nseq * s->width * 4);
        };
        bool again = same(in) || same(out);
        for (int64_t j = 0; j < i; ++j) again |= same(others[j]);
        if (again) return report(VS_ERR_INVALID, "other %lld is named twice", (long long)i);
    }
    vs::DeviceGuard g(kv->device);
    if (g.err != hipSuccess) return report_hip(g.err, "hipSetDevice");
    hipStream_t st = (hipStream_t)stream;
    const int64_t np = kv->npages;
    void *ws = nullptr;
    rc = kv->scratch.get(st, (size_t)(3 * np + 1) * sizeof(int32_t), &ws);
    if (rc) return rc;
    vs::CompactArgs a = {};
    a.refs = in->refs;
    a.refs2 = out->refs;
    a.npages = (int)np;
    a.map = map ? map : (int32_t *)ws;
    a.from = (int32_t *)ws + np;
    a.to = a.from + np;
    a.moves = a.to + np;
    a.status = kv->status;
    a.closed = kv->closed;
    if (np <= vs::kSmallPages)
        hipLaunchKernelGGL(vs::compact_plan_small_kernel, dim3(1), dim3(vs::kPlan), 0, st, a);
    else
        hipLaunchKernelGGL(vs::compact_plan_kernel, dim3(1), dim3(vs::kPlan), 0, st, a);
    VS_LAUNCHED("compact");
    const vs::Tables tables = {in->table,  in->lens,  a.map,
                               out->table, out->lens, in->nseq * in->width,
                               (int)in->nseq};
    hipError_t e = vs::launch_copy(kv, a.moves, np / 2 + 1, a.from, a.to, 1, st, tables);
    if (e != hipSuccess) return report_hip(e, "page copies");
    for (int64_t i = 0; i < nothers; ++i) {
        const int64_t entries = others[i]->nseq * others[i]->width;
        if (!entries) continue;
        hipLaunchKernelGGL(vs::remap_kernel, dim3(vs::grid_of((entries + 255) / 256, 2048)), dim3(256),
                           0, st, others[i]->table, entries, (int)np, a.map);
        VS_LAUNCHED("compact");
    }
    return VS_OK;
}

int vs_kv_copy(vs_kv *kv, const int32_t *from, const int32_t *to, int64_t n, void *stream) {
    if (!kv) return report(VS_ERR_INVALID, "null handle");
    if (n < 0) return report(VS_ERR_INVALID, "n %lld", (long long)n);
    if (n == 0) return VS_OK;
    if (!from || !to || ((uintptr_t)from | (uintptr_t)to) % 4)
        return report(VS_ERR_INVALID, "null or unaligned page lists");
    vs::DeviceGuard g(kv->device);
    if (g.err != hipSuccess) return report_hip(g.err, "hipSetDevice");
    hipError_t e = vs::launch_copy(kv, nullptr, n, from, to, 1, (hipStream_t)stream);
    return e == hipSuccess ? VS_OK : report_hip(e, "page copies");
}

int vs_kv_check(vs_kv *kv, void *stream) {
    if (!kv) return report(VS_ERR_INVALID, "null handle");
    vs::DeviceGuard g(kv->device);
    if (g.err != hipSuccess) return report_hip(g.err, "hipSetDevice");
    hipStream_t st = (hipStream_t)stream;
    int32_t got[vs::kStatusWords] = {0};
    hipError_t e = hipStreamSynchronize(st);
    if (e == hipSuccess) e = hipMemcpy(got, kv->status, sizeof got, hipMemcpyDeviceToHost);
    if (e == hipSuccess && got[2]) {
        // what other streams still run behind a refused extend must find its pages closed
        e = hipDeviceSynchronize();
        if (e == hipSuccess) e = hipMemcpy(got, kv->status, sizeof got, hipMemcpyDeviceToHost);
        if (e == hipSuccess) e = hipMemset(kv->closed, 0, (size_t)kv->npages);
    }
    if (e == hipSuccess && got[0]) e = hipMemset(kv->status, 0, sizeof got);
    if (e == hipSuccess && got[0]) e = hipStreamSynchronize(nullptr);
    if (e != hipSuccess) return report_hip(e, "check");
    if (got[0] & vs::kStatusPages)
        return report(VS_ERR_OOM, "the cache was %d pages short", (int)got[1]);
    if (got[0] & vs::kStatusWidth)
        return report(VS_ERR_INVALID, "a sequence outgrew its %s", "table row");
    if (got[0] & vs::kStatusNoPage) return report(VS_ERR_INVALID, "a new token has no page");
    if (got[0] & vs::kStatusParent) return report(VS_ERR_INVALID, "a parent is out of range");
    return VS_OK;
}

}  // extern "C"

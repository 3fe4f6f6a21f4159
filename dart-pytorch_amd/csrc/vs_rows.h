// vs_rows.h -- rows of queries, keys and values beside the paged cache, shared by
// the sources of its attention, its rotary positions and its rows in and out.
#pragma once

#include "vs_kv.h"

namespace vs {

// 16 bytes of a row from element x on, whatever the row's alignment.
template <int ST>
__device__ __forceinline__ u32x4_t load_piece(const char *row, int x, bool vec) {
    constexpr int E = ST ? 8 : 4;
    if (vec) return *(const u32x4_t *)(row + (int64_t)x * (16 / E));
    u32x4_t w;
    if constexpr (ST) {
        const uint16_t *p = (const uint16_t *)row + x;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (uint32_t)p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
    } else {
        const uint32_t *p = (const uint32_t *)row + x;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = p[i];
    }
    return w;
}

// The place of position t of a block, dimension x, in elements.
template <int ST>
__host__ __device__ inline int key_place(int t, int x, int dim) {
    constexpr int E = ST ? 8 : 4;
    return ((t / 16 * (dim / E) + x / E) * 16 + t % 16) * E + x % E;
}
template <int ST>
__host__ __device__ inline int value_place(int t, int x, int dim) {
    const int h = t / 16, g = t % 16 / 4, i = t % 4;
    return ST ? ((x * 4 + g) * 2 + h) * 4 + i : ((h * dim + x) * 4 + g) * 4 + i;
}

struct RowsArgs {
    char *pool;
    int64_t page_bytes, layer_off, kv_off, head_off;
    const int32_t *table, *lens, *starts;
    int64_t width, nrows;
    int nseq, npages, page_shift, heads, dim;
    int32_t *status;
    const uint8_t *closed;
    const char *k, *v;
    int64_t k_row, k_head, v_row, v_head;
    int k_vec, v_vec;  // rows readable in 16-byte pieces
    char *k_out, *v_out;
    int b, first;
};

// Where position pos of sequence b lies; null if nowhere.
__device__ __forceinline__ char *block_of(const RowsArgs &a, int b, int64_t pos, int es) {
    if (pos < 0 || pos >> a.page_shift >= a.width) return nullptr;
    const int page = a.table[(int64_t)b * a.width + (pos >> a.page_shift)];
    if ((unsigned)page >= (unsigned)a.npages) return nullptr;
    const int64_t blk = (pos & ((1 << a.page_shift) - 1)) / kKvBlock;
    return a.pool + (int64_t)page * a.page_bytes + a.layer_off + blk * kKvBlock * a.dim * es;
}

// A block's values from LDS (a row of ld elements per position) to their places:
// positions t0 <= t < t1, in whole pieces where all of a piece's are.
template <int ST, typename T>
__device__ __forceinline__ void store_values(const T *rows, int ld, T *to, int dim, int t0, int t1) {
    constexpr int E = ST ? 8 : 4;
    for (int x = threadIdx.x; x < kKvBlock * dim / E; x += 256) {
        // bf16: [dimension][g][half][i], fp32: [half][dimension][g][i]
        const int g = x % 4, d = ST ? x / 4 : x / 4 % dim, half = ST ? 0 : x / 4 / dim;
        T out[E];
        int have = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int t = 16 * (ST ? e / 4 : half) + 4 * g + e % 4;
            const bool in = t >= t0 && t < t1;
            out[e] = in ? rows[t * ld + d] : (T)0;
            have += in;
        }
        T *dst = to + x * E;
        if (have == E) {
            u32x4_t v;
            __builtin_memcpy(&v, out, 16);
            *(u32x4_t *)dst = v;
        } else if (have) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int t = 16 * (ST ? e / 4 : half) + 4 * g + e % 4;
                if (t >= t0 && t < t1) dst[e] = out[e];
            }
        }
    }
}

// The last of n ascending values (value(i), i < n) that is at or below x, or 0:
// the wave's lanes look at 64 of them at once.
template <typename F>
__device__ __forceinline__ int64_t last_at_or_below(int64_t n, int64_t x, int lane, F value) {
    int64_t lo = 0;  // it is one of lo .. lo + n - 1
    while (n > 1) {
        const int64_t step = (n + 63) / 64, i = lo + lane * step;
        const uint64_t in = __ballot(lane * step < n && value(i) <= x);
        const int l = in ? 63 - __builtin_clzll(in) : 0;
        lo += l * step;
        n = min(step, n - l * step);
    }
    return lo;
}

// Where a layer's heads lie in a page, in bytes.
template <typename Args>
inline void fill_geometry(const vs_kv *kv, int64_t layer, Args &a) {
    const int64_t e = kv_elem(kv->dtype);
    a.pool = kv->mem;
    a.page_bytes = kv->page_bytes;
    a.head_off = kv->page_size * kv->head_dim * e;
    a.kv_off = kv->kv_heads * a.head_off;
    a.layer_off = layer * 2 * a.kv_off;
}

// |stride| elements of n rows and of heads stay inside 2^62 bytes
inline bool stride_ok(int64_t s, int64_t n = 1 << 20) {
    const int64_t most = ((int64_t)1 << 60) / std::clamp<int64_t>(n, 1 << 20, INT32_MAX);
    return s >= -most && s <= most;
}

inline bool pieces_ok(const void *p, int64_t s0, int64_t s1, int64_t e) {
    return (((uintptr_t)p | (uintptr_t)(s0 * e) | (uintptr_t)(s1 * e)) & 15) == 0;
}

// Whether an output shares a byte with what tells the kernels where rows go.
inline bool over_places(const Extent &out, const vs_kv_seqs *s, const int32_t *starts) {
    auto shares = [&](const int32_t *p, int64_t n) { return p && n > 0 && meet(out, Extent(p, 0, 0, 1, 1, n, 4)); };
    return shares(starts, s->nseq + 1) || shares(s->lens, s->nseq) || shares(s->table, s->nseq * s->width);
}

inline int fill_rows(const vs_kv *kv, const vs_kv_seqs *s, int64_t layer, RowsArgs &a) {
    if (layer < 0 || layer >= kv->layers)
        return report(VS_ERR_INVALID, "layer %lld out of range [0, %lld)", (long long)layer,
                      (long long)kv->layers);
    fill_geometry(kv, layer, a);
    a.table = s->table;
    a.lens = s->lens;
    a.width = s->width;
    a.nseq = (int)s->nseq;
    a.npages = (int)kv->npages;
    a.status = kv->status;
    a.closed = kv->closed;
    a.page_shift = __builtin_ctzll((uint64_t)kv->page_size);
    a.heads = (int)kv->kv_heads;
    a.dim = (int)kv->head_dim;
    return VS_OK;
}

}  // namespace vs

// vs_attend.hip -- attention of one new token over the paged key-value cache,
// and the cache's rows in and out: kernels and entry points.
#include <cmath>

#include "vs_device.h"
#include "vs_rows.h"
#include "vs_wave.h"

namespace vs {
namespace {

constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kWaves = 4;      // per workgroup
constexpr int kMinBlocks = 4;  // blocks per work item, at least: one per wave
constexpr int kGoodBlocks = 8; // and before a CU takes a second workgroup
constexpr int kFindSeqs = 384; // sequences that each workgroup divides for itself
// dimensions joined over the waves at once, by what LDS holds
constexpr int join_dims(int waves) { return waves == 8 ? 64 : 128; }
constexpr int kWideDim = 128;  // heads up to this size have an eight-wave kernel

struct AttendArgs {
    char *pool;
    int64_t page_bytes, layer_off, kv_off, head_off;  // bytes; kv_off from keys to values
    const int32_t *table, *lens;
    int64_t width;
    int nseq, npages, page_shift;
    const char *q, *k, *v;
    char *out;
    int64_t q_seq, q_head, k_seq, k_head, v_seq, v_head, o_seq, o_head;  // elements
    float *lse;
    int heads, kv_heads, group, gtiles;  // group: query heads per key-value head; gtiles: 16 at a time
    float scale2;                        // scale * log2(e)
    int window, sinks;
    int unsplit;                         // one item per sequence
    int q_vec, k_vec;                    // rows readable in 16-byte pieces
    int most_items, few_items;           // six workgroups to a CU, and one
    float *part_o;   // [item][heads][dim]
    float2 *part_ml; // [item][heads] running maximum and sum
    int32_t *status;
    const uint8_t *closed;
    int2 *first;     // [nseq] first whole item; whole ones * 2 + whether there is a rest
    int32_t *plan;   // blocks per piece, then [item] its sequence, or -1; null: find_item
    int items;
};

// The blocks that a sequence of n positions attends to: nsb from its start,
// then wb0 .. nb - 1.
struct Span {
    int nsb, wb0, total;
};

__device__ __forceinline__ Span span_of(int n, int window, int sinks) {
    Span s;
    const int nb = n / kKvBlock + (n % kKvBlock != 0);
    s.nsb = s.wb0 = 0;
    if (window > 0 && n > window) {
        s.wb0 = (n - window) / kKvBlock;
        const int k = min(sinks, n);
        s.nsb = min(k / kKvBlock + (k % kKvBlock != 0), s.wb0);
    }
    s.total = s.nsb + nb - s.wb0;
    return s;
}

__device__ __forceinline__ int length_of(const AttendArgs &a, int b) {
    const int64_t most = a.width << a.page_shift;
    const int n = max(a.lens[b], 0);
    return n < most ? n : (int)most;
}

// Blocks of sequence b.
__device__ __forceinline__ int blocks_of(const AttendArgs &a, int b) {
    return span_of(length_of(a, b), a.window, a.sinks).total;
}

// How many blocks a piece has: `total` of all sequences, `widest` of one.
// Lengths far apart: pieces a third as long, which spread better (64
// sequences of 65 to 8,190 positions 98 against 107 us, 256 of 100 to 4,000
// 128 against 139); about equal ones: as few joins as can be (64 of 4,096
// 191 against 196 us).
__device__ __forceinline__ int blocks_per_piece(const AttendArgs &a, uint64_t total, int widest) {
    auto over = [&](int items) {
        return total >> 31 ? (int)((total + items - 1) / (uint64_t)items)
                           : (int)(((uint32_t)total + items - 1) / (uint32_t)items);
    };
    const bool ragged = (uint64_t)widest * a.nseq > 2 * total;
    const int items = max(ragged ? a.most_items : a.most_items / 3, 1);
    int per = max(max(over(items), min(over(a.few_items), kGoodBlocks)), kMinBlocks);
    // (and equal ones: a small rest of every sequence would be a workgroup more each)
    if (!ragged && widest > per) {
        int pieces = (widest + per - 1) / per;
        if ((uint64_t)pieces * a.nseq > (uint64_t)items) pieces = widest / per;
        per = (widest + pieces - 1) / pieces;
    }
    return per;
}

// Work item `item`: blocks [split * per, ...) of sequence b.  Every wave works
// the division out by itself from the lengths (of up to kFindSeqs sequences: the
// work is that of all lengths per workgroup).  `per` is all blocks of the
// call over the workgroups that the card holds at once, so that long sequences
// of a ragged batch are split and short ones are not.  First come all whole
// pieces of `per` blocks, then what is left of the sequences: the smaller ones
// fill the places that come free.  There are no gaps in the numbers: a
// workgroup that finds no work does not give its place to the next (one
// sequence of 100,000 positions 82 against 72 us).
struct Item {
    int b, split, per;
    int first, whole, rest;  // the sequence's pieces: items first .. first + whole - 1, and a rest
};

__device__ __forceinline__ bool find_item(const AttendArgs &a, int item, int lane, Item &it) {
    auto blocks = [&](int b) { return b < a.nseq ? blocks_of(a, b) : -1; };
    const int t0 = blocks(lane);  // (all there is to read for up to 64 sequences)
    uint64_t mine = max(t0, 0);
    int widest = max(t0, 0);
    for (int b = lane + 64; b < a.nseq; b += 64) {
        const int t = blocks(b);
        mine += (uint64_t)t;
        widest = max(widest, t);
    }
    // (2^20 sequences of 2^26 blocks at most)
    const uint64_t total = ((uint64_t)wave_sum((uint32_t)(mine >> 20)) << 20) +
                           wave_sum((uint32_t)mine & 0xFFFFF);
    // (past 2^24 blocks a float is off by two of them at most, less than a piece)
    const int per = blocks_per_piece(a, total, (int)wave_max((float)widest));
    it.per = per;
    int wholes = 0;
    for (int b0 = 0; b0 < a.nseq; b0 += 64)
        wholes += (int)wave_sum((uint32_t)max(b0 ? blocks(b0 + lane) : t0, 0) / (uint32_t)per);
    // the sequence whose whole pieces, or whose rest, the item's number falls into
    const bool rest_item = item >= wholes;
    int base = 0, rank = wholes;
    for (int b0 = 0; b0 < a.nseq; b0 += 64) {
        const int t = b0 ? blocks(b0 + lane) : t0;
        const int whole = (int)((uint32_t)max(t, 0) / (uint32_t)per);
        // (a sequence without blocks has its empty answer to write)
        const int rest = t >= 0 && (t == 0 || t != whole * per);
        const int wsum = base + prefix_sum(whole), rsum = rank + prefix_sum(rest);
        const uint64_t past = __ballot(rest_item ? rsum > item : wsum > item);
        if (past) {
            const int l = __builtin_ctzll(past);
            it.b = b0 + l;
            it.whole = __builtin_amdgcn_readlane(whole, l);
            it.rest = __builtin_amdgcn_readlane(rest, l);
            it.first = __builtin_amdgcn_readlane(wsum, l) - it.whole;
            it.split = rest_item ? it.whole : item - it.first;
            return true;
        }
        base = __builtin_amdgcn_readlane(wsum, 63);
        rank = __builtin_amdgcn_readlane(rsum, 63);
    }
    return false;
}

// The same division as find_item's, once for all workgroups of the call: a launch
// and 9 us, but each workgroup then has three loads instead of all lengths to
// read.  find_item against this, 8 key-value heads of 128 in bf16, lengths of 64 to
// 3,000 (and of 64 but for one of 16,384): 256 sequences 127 and 133 us (45 and 45),
// 384 184 and 187 (63 and 51), 512 242 and 241 (85 and 58), 1,024 491 and 460, 4,096
// 2,975 and 1,802, 16,384 32,600 and 7,020.  With 1 head 256 30 and 36, 512 52 and
// 51, 4,096 483 and 270.
__global__ __launch_bounds__(kPlan) void attend_plan_kernel(AttendArgs a) {
    __shared__ int lds[kPlan / 64];
    __shared__ unsigned long long sum;
    __shared__ int most;
    if (threadIdx.x == 0) {
        sum = 0;
        most = 0;
    }
    uint64_t mine = 0;
    int widest = 0;
    for (int b = threadIdx.x; b < a.nseq; b += kPlan) {
        const int t = blocks_of(a, b);
        mine += (uint64_t)t;
        widest = max(widest, t);
    }
    __syncthreads();
    atomicAdd(&sum, (unsigned long long)mine);
    atomicMax(&most, widest);
    __syncthreads();
    const int per = blocks_per_piece(a, sum, most);
    int32_t *seq_of = a.plan + 1;
    int base = 0, total;
    for (int b0 = 0; b0 < a.nseq; b0 += kPlan) {
        const int b = b0 + threadIdx.x, t = b < a.nseq ? blocks_of(a, b) : 0;
        const int whole = (int)((uint32_t)t / (uint32_t)per);
        const int at = base + block_scan(whole, &total, lds);
        base += total;
        if (b >= a.nseq) continue;
        a.first[b] = make_int2(at, whole * 2 + (t == 0 || t != whole * per));
        for (int i = 0; i < whole; ++i) seq_of[at + i] = b;
    }
    for (int b0 = 0; b0 < a.nseq; b0 += kPlan) {
        const int b = b0 + threadIdx.x;
        const int rest = b < a.nseq ? a.first[b].y & 1 : 0;  // (its own store)
        const int at = base + block_scan(rest, &total, lds);
        base += total;
        if (rest) seq_of[at] = b;
    }
    for (int i = base + threadIdx.x; i < a.items; i += kPlan) seq_of[i] = -1;
    if (threadIdx.x == 0) a.plan[0] = per;
}

// The larger of the four lanes that share a column (lanes apart by 16).
__device__ __forceinline__ float column_max(float x) {
    typedef unsigned u32pair __attribute__((ext_vector_type(2)));
    u32pair p = __builtin_amdgcn_permlane16_swap(bits_of(x), bits_of(x), false, false);
    x = fmaxf(float_of(p.x), float_of(p.y));
    p = __builtin_amdgcn_permlane32_swap(bits_of(x), bits_of(x), false, false);
    return fmaxf(float_of(p.x), float_of(p.y));
}

// One pass over a work item's keys and values with the running maximum and
// sum of the softmax.  A wave takes every fourth unit of the item: 32
// positions of bf16, 16 of fp32.  Lane (r, g) = (lane & 15, lane >> 4).
//   S^T = K Q^T    A operand: key rows (position r, 16 bytes of dimensions g);
//                  B operand: the query heads of the group, column r
//   O^T = V^T P^T  A operand: dimension r, the positions of lane group g;
//                  B operand: P^T, which is S^T's accumulator as it stands:
//                  lane (r, g) holds query r at positions 16 h + 4 g + i, and
//                  the values lie in the cache in that order
// so nothing passes through LDS but the join of the four waves, every load is
// 1 KB of consecutive bytes per wave, and a column's maximum, sum and
// rescaling belong to one lane.  Unused columns (fewer than 16 query heads
// per key-value head) cost matrix time that the loads leave idle anyway.
// bf16: P is multiplied as the sum of three bf16 values, its 24 bits eight at a
// time, so the output is that of 32-bit weights, rounded once.  (Two of them, 16
// bits, sent two to four answers in a thousand to the other neighbour.)  The
// third product costs 0 to 2 % (head sizes 32 to 256, 64 sequences of 2,000:
// 25.7 to 26.1 us at 32, 102.7 to 103.0 at 128), because each part is split off
// after the one before is multiplied: all three at once took 12 to 30 registers
// and a wave per SIMD more (head size 32, 64 ragged ones 19.7 against 18.1 us).
//
// Bound by HBM: each byte of the cache is read once per 16 query heads.  8
// key-value heads of 128 in bf16: 2 sequences of 120,000 to 131,000 positions
// 176 us (1.03 GB, 5.9 TB/s of the 6.3 that a plain read reaches), 64 of 65 to
// 8,190 93 us (470 MB, 5.0 TB/s: the spread of the pieces' ends).  One of 1,000
// is bound by latency, 7 us.
//
// In the loop a unit's keys are replaced by the next one's as soon as they are
// multiplied, and so are its values: loads are in flight all the time.
// NW waves: four, or eight where short sequences are not split and a workgroup
// has a whole one (a.unsplit).
template <int ST, int D, int NW>
__global__ __launch_bounds__(64 * NW, D <= 96 ? 3 : NW == 8 || D <= (ST ? 192 : 160) ? 2 : 1)
    void attend_kernel(AttendArgs a) {
    constexpr int E = ST ? 8 : 4;
    constexpr int ES = 16 / E;             // element size
    constexpr int H = ST ? 2 : 1;          // 16-position halves per unit
    constexpr int UB = ST ? 1 : 2;         // units per block
    constexpr int NC = (D / E + 3) / 4;    // 16-byte pieces per lane of a key row
    constexpr int ND = D / 16;
    constexpr int DW = D < join_dims(NW) ? D : join_dims(NW);
    constexpr int LD = DW + 4;
    constexpr float kNone = -__builtin_huge_valf();
    extern __shared__ __align__(16) float lds_o[];  // [wave][query][LD]
    __shared__ float lds_m[NW][16], lds_l[NW][16];
    __shared__ u32x4_t lds_k[D / E];  // the new token
    __shared__ uint32_t lds_v[D];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int per_item = a.kv_heads * a.gtiles;
    const int item = blockIdx.x / per_item, hh = blockIdx.x % per_item;
    const int gt = hh / a.kv_heads, kvh = hh % a.kv_heads;
    const int gc = min(a.group - gt * 16, 16);  // query heads of this workgroup
    // some page may take no new token (loaded here, to be back when that counts)
    const int marked = a.status[2];
    Item it = {};
    if (a.unsplit) {
        it.b = item;
        it.per = INT32_MAX / kKvBlock;
        it.rest = 1;
    } else if (a.plan) {
        it.b = __builtin_amdgcn_readfirstlane(a.plan[1 + item]);
        if (it.b < 0) return;
        it.per = __builtin_amdgcn_readfirstlane(a.plan[0]);
        it.first = __builtin_amdgcn_readfirstlane(a.first[it.b].x);
        const int pieces = __builtin_amdgcn_readfirstlane(a.first[it.b].y);
        it.whole = pieces >> 1;
        it.rest = pieces & 1;
        // (the rests' numbers come behind all whole ones)
        it.split = min(item - it.first, it.whole);
    } else if (!find_item(a, item, lane, it)) {
        return;
    }
    const int n = __builtin_amdgcn_readfirstlane(length_of(a, it.b));
    const Span sp = span_of(n, a.window, a.sinks);
    const int head0 = kvh * a.group + gt * 16;

    // the queries, as the B operand
    u32x4_t qf[NC];
    {
        const char *row = a.q + ((int64_t)it.b * a.q_seq + (int64_t)(head0 + r) * a.q_head) * ES;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            qf[c] = u32x4_t{0, 0, 0, 0};
            if (r < gc && c * 4 + g < D / E) qf[c] = load_piece<ST>(row, (c * 4 + g) * E, a.q_vec);
        }
    }

    float m = kNone, l = 0.f;
    f32x4_t o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    const int32_t *trow = a.table + (int64_t)it.b * a.width;
    char *const head_base = a.pool + a.layer_off + (int64_t)kvh * a.head_off;
    const int bpp1 = (1 << (a.page_shift - 5)) - 1;
    const int j0 = it.split * it.per, j1 = min(j0 + it.per, sp.total);
    // first position of unit u, counted along the span
    auto unit_pos = [&](int u) {
        const int j = u / UB;
        return (j < sp.nsb ? j : j - sp.nsb + sp.wb0) * kKvBlock + u % UB * 16;
    };
    auto unit_keys = [&](int page, int pos) {
        return head_base + (int64_t)page * a.page_bytes +
               (((pos >> 5) & bpp1) * kKvBlock + (pos & 16)) * (D * ES);
    };
    // blocks with a mask in them
    const bool cut = a.window > 0 && n > a.window;
    auto edge = [&](int j) {
        return j == sp.total - 1 || (cut && (j == sp.nsb || j == sp.nsb - 1));
    };
    u32x4_t kf[H * NC], vf[ND];
    auto load_keys = [&](const char *kb) {
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                // (a piece past the row's end is read again and zeroed)
                const int piece = D % (4 * E) ? min(c * 4 + g, D / E - 1) : c * 4 + g;
                kf[h * NC + c] = *(const u32x4_t *)(kb + ((h * (D / E) + piece) * 16 + r) * 16);
            }
    };
    auto load_values = [&](const char *kb) {
#pragma unroll
        for (int d = 0; d < ND; ++d)
            vf[d] = *(const u32x4_t *)(kb + a.kv_off + ((d * 16 + r) * 4 + g) * 16);
    };
    f32x4_t s[H];
    auto scores = [&]() {
#pragma unroll
        for (int h = 0; h < H; ++h) {
            if constexpr (D % (4 * E) != 0) {
                if ((NC - 1) * 4 + g >= D / E) kf[h * NC + NC - 1] = u32x4_t{0, 0, 0, 0};
            }
            s[h] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                if constexpr (ST) {
                    s[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        __builtin_bit_cast(bf16x8_t, kf[h * NC + c]),
                        __builtin_bit_cast(bf16x8_t, qf[c]), s[h], 0, 0, 0);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                            float_of(kf[h * NC + c][e]), float_of(qf[c][e]), s[h], 0, 0, 0);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) s[h][i] *= a.scale2;
        }
    };
    auto weigh = [&]() {
        float top = s[0][0];
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, s[h][i]);
        top = column_max(top);
        if (__ballot(top > m)) {
            const float mn = fmaxf(m, top);
            const float f = mn == m ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= f;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[d][i] *= f;
        }
        const float ms = m == kNone ? 0.f : m;
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[h][i] = __builtin_amdgcn_exp2f(s[h][i] - ms);
                l += s[h][i];
            }
    };
    auto add_values = [&]() {
        if constexpr (ST) {
#pragma unroll
            for (int j = 0; j < 3; ++j) {
                bf16x8_t part;
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float t = float_of(bits_of(s[h][i]) & 0xFFFF0000u);
                        // (the rest is never 0 beside a weight: an infinite value times
                        // 0 would be a NaN)
                        if (j < 2) s[h][i] = fmaxf(s[h][i] - t, t * 0x1p-30f);
                        part[4 * h + i] = (__bf16)t;
                    }
#pragma unroll
                for (int d = 0; d < ND; ++d)
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        __builtin_bit_cast(bf16x8_t, vf[d]), part, o[d], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int d = 0; d < ND; ++d)
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(float_of(vf[d][i]), s[0][i], o[d],
                                                                0, 0, 0);
        }
    };

    // The wave's units in order: 64 at a time, lane i looks the page of the i-th
    // up, and those that have one are a bit mask.
    const int u0 = j0 * UB + wave, count = max((j1 * UB - u0 + NW - 1) / NW, 0);
    int chunk = -64, pages = -1;
    uint64_t ready = 0;
    int u_n = 0;  // the unit found, and its keys
    const char *kb_n = a.pool;
    auto next_unit = [&]() {
        while (!ready) {
            chunk += 64;
            if (chunk >= count) return false;
            pages = -1;
            if (chunk + lane < count)
                pages = trow[unit_pos(u0 + (chunk + lane) * NW) >> a.page_shift];
            ready = __ballot((unsigned)pages < (unsigned)a.npages);
        }
        const int i = __builtin_ctzll(ready);
        ready &= ready - 1;
        u_n = u0 + (chunk + i) * NW;
        kb_n = unit_keys(__builtin_amdgcn_readlane(pages, i), unit_pos(u_n));
        return true;
    };

    // The new token, at position n - 1: read before all else and laid down in
    // LDS, so that no load of it is waited for at the end.
    int u_new = -1, t_new = 0;  // the unit that holds it, if it is the wave's, and its place there
    u32x4_t k_new = {0, 0, 0, 0};
    uint32_t v_new[(D + 63) / 64];
    int new_page = -1;
    if (a.k && sp.total > 0) {
        t_new = (n - 1) % (16 * H);
        const int u = (sp.total - 1) * UB + (n - 1) % kKvBlock / (16 * H);
        if (u >= u0 && u < j1 * UB && (u - u0) % NW == 0) {
            new_page = trow[(n - 1) >> a.page_shift];
            if (a.lens[it.b] > n) {  // past the table: n - 1 is not the new token's place
                if (lane == 0) atomicOr(&a.status[0], kStatusWidth);
            } else if ((unsigned)new_page >= (unsigned)a.npages) {
                if (lane == 0) atomicOr(&a.status[0], kStatusNoPage);
            } else if (!(marked && a.closed[new_page])) {
                u_new = u;
            }
        }
    }
    if (u_new >= 0) {
        const char *krow = a.k + ((int64_t)it.b * a.k_seq + (int64_t)kvh * a.k_head) * ES;
        const char *vrow = a.v + ((int64_t)it.b * a.v_seq + (int64_t)kvh * a.v_head) * ES;
        if (lane < D / E) k_new = load_piece<ST>(krow, lane * E, a.k_vec);
#pragma unroll
        for (int i = 0; i < (D + 63) / 64; ++i) {
            const int x = min(lane + 64 * i, D - 1);
            v_new[i] = ST ? ((const uint16_t *)vrow)[x] : ((const uint32_t *)vrow)[x];
        }
    }
    bool more = next_unit();
    const bool any = more;
    if (any) {
        load_keys(kb_n);
        load_values(kb_n);
    }
    if (u_new >= 0) {
        if (lane < D / E) lds_k[lane] = k_new;
#pragma unroll
        for (int i = 0; i < (D + 63) / 64; ++i)
            if (lane + 64 * i < D) lds_v[lane + 64 * i] = v_new[i];
        lds_wave_sync();
    }
    if (any) {
        int u;
        do {
            u = u_n;
            more = next_unit();
            // (loads under a condition would be waited for as if those behind
            // them had not been issued: the last unit reads some page again)
            const char *kb = more ? kb_n : head_base;
            if (u == u_new) {
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int c = 0; c < NC; ++c)
                        if (t_new == 16 * h + r && c * 4 + g < D / E)
                            kf[h * NC + c] = lds_k[c * 4 + g];
                // stored with its neighbours, in whole cache lines
                if (gt == 0) {
                    char *to = unit_keys(new_page, unit_pos(u));
#pragma unroll
                    for (int h = 0; h < H; ++h)
#pragma unroll
                        for (int c = 0; c < NC; ++c)
                            if (t_new / 16 == h && c * 4 + g < D / E)
                                *(u32x4_t *)(to + ((h * (D / E) + c * 4 + g) * 16 + r) * 16) =
                                    kf[h * NC + c];
                }
            }
            scores();
            load_keys(kb);
            if (u == u_new) {
                const bool mine = (t_new & 15) >> 2 == g;
                const int at = (t_new >> 4) * 4 + (t_new & 3);  // its element of the lane's 16 bytes
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const uint32_t x = lds_v[d * 16 + r];
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        if constexpr (ST) {
                            if (mine && w == at >> 1)
                                vf[d][w] = at & 1 ? (vf[d][w] & 0xFFFFu) | x << 16
                                                  : (vf[d][w] & 0xFFFF0000u) | x;
                        } else {
                            if (mine && w == at) vf[d][w] = x;
                        }
                    }
                }
                if (gt == 0) {
                    char *to = unit_keys(new_page, unit_pos(u)) + a.kv_off;
#pragma unroll
                    for (int d = 0; d < ND; ++d)
                        *(u32x4_t *)(to + ((d * 16 + r) * 4 + g) * 16) = vf[d];
                }
            }
            if (edge(u / UB)) {
                // a masked position's score is -inf and its values are 0: what
                // lies there may be anything, and 0 times a NaN is one
                const int pos0 = unit_pos(u);
                const int low = a.window > 0 ? n - a.window : 0;  // below, only sinks are visible
                uint32_t hide = 0;
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int p = pos0 + 16 * h + 4 * g + i;
                        if (p >= n || (p < low && p >= a.sinks)) {
                            s[h][i] = kNone;
                            hide |= 1u << (4 * h + i);
                        }
                    }
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t keep = ~0u;
                    if constexpr (ST) {
                        if (hide >> (2 * w) & 1) keep &= 0xFFFF0000u;
                        if (hide >> (2 * w + 1) & 1) keep &= 0x0000FFFFu;
                    } else {
                        if (hide >> w & 1) keep = 0;
                    }
#pragma unroll
                    for (int d = 0; d < ND; ++d) vf[d][w] &= keep;
                }
            }
            weigh();
            add_values();
            load_values(kb);
        } while (more);
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) {
        lds_m[wave][r] = m;
        lds_l[wave][r] = l;
    }

    // the waves' sums, DW dimensions at a time
    const bool last = it.whole + it.rest <= 1;
#pragma unroll
    for (int d0 = 0; d0 < ND; d0 += DW / 16) {
        if (d0) __syncthreads();
        if (r < gc)
#pragma unroll
            for (int d = 0; d < DW / 16; ++d)
                if (d0 + d < ND)
                    *(f32x4_t *)(lds_o + (wave * gc + r) * LD + d * 16 + g * 4) = o[d0 + d];
        __syncthreads();
        const int dims = min(DW, D - d0 * 16);
        for (int x = threadIdx.x; x < gc * (DW / 4); x += 64 * NW) {
            const int row = x / (DW / 4), c4 = x % (DW / 4);
            if (c4 * 4 >= dims) continue;
            float top = lds_m[0][row];
#pragma unroll
            for (int w = 1; w < NW; ++w) top = fmaxf(top, lds_m[w][row]);
            const float ms = top == kNone ? 0.f : top;
            float sum = 0.f;
            f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float f = __builtin_amdgcn_exp2f(lds_m[w][row] - ms);
                sum += f * lds_l[w][row];
                const f32x4_t t = *(const f32x4_t *)(lds_o + (w * gc + row) * LD + c4 * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i] += f * t[i];
            }
            const int head = head0 + row, dim = d0 * 16 + c4 * 4;
            if (last) {
                char *to = a.out + ((int64_t)it.b * a.o_seq + (int64_t)head * a.o_head + dim) * ES;
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (ST)
                        ((__bf16 *)to)[i] = (__bf16)(acc[i] * inv);
                    else
                        ((float *)to)[i] = acc[i] * inv;
                }
                if (a.lse && dim == 0)
                    a.lse[(int64_t)it.b * a.heads + head] =
                        sum == 0.f ? kNone : (top + __builtin_amdgcn_logf(sum)) * kLn2;
            } else {
                const int64_t slot =
                    (int64_t)(it.split < it.whole ? item : a.most_items + it.b) * a.heads + head;
                *(f32x4_t *)(a.part_o + slot * D + dim) = acc;
                if (dim == 0) a.part_ml[slot] = make_float2(top, sum);
            }
        }
    }
    if (a.first && !a.plan && hh == 0 && it.split == 0 && threadIdx.x == 0)
        a.first[it.b] = make_int2(it.first, it.whole * 2 + it.rest);
}

// Joins the items of a sequence, in their order: one workgroup per query head,
// its waves taking every fourth item.  Bound by two loads that follow each
// other and the launch: 2.5 to 5 us.  (The workgroup that is done last could
// do it and save the launch; but the fences that this needs between the L2
// caches, one per workgroup, took longer: 16 sequences of 4,096 positions 76
// against 58 us.)
template <int ST, int D>
__global__ __launch_bounds__(64 * kWaves) void attend_join_kernel(AttendArgs a) {
    constexpr int NR = (D + 63) / 64;
    constexpr int ES = ST ? 2 : 4;
    constexpr float kNone = -__builtin_huge_valf();
    __shared__ float lds_a[kWaves][NR * 64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.x / a.heads, head = blockIdx.x % a.heads;
    const int2 f = a.first[b];
    const int whole = f.y >> 1, cnt = whole + (f.y & 1);
    if (cnt <= 1) return;
    auto slot_of = [&](int s) {
        return (int64_t)(s < whole ? f.x + s : a.most_items + b) * a.heads + head;
    };
    // eight of the wave's partial sums at a time, the first ones in flight while
    // the maximum and the sum over all items are found (by every wave)
    float t[8][NR], w[8], acc[NR];
    auto load = [&](int s0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int64_t slot = slot_of(min(s0 + e * kWaves, cnt - 1));
            w[e] = a.part_ml[slot].x;
#pragma unroll
            for (int i = 0; i < NR; ++i)
                t[e][i] = a.part_o[slot * D + min(lane + 64 * i, D - 1)];
        }
    };
    load(wave);
    float top = kNone, sum = 0.f;
    for (int s = lane; s < cnt; s += 64) {
        const float2 ml = a.part_ml[slot_of(s)];
        const float mn = fmaxf(top, ml.x);
        const float ms = mn == kNone ? 0.f : mn;
        sum = sum * __builtin_amdgcn_exp2f(top - ms) + ml.y * __builtin_amdgcn_exp2f(ml.x - ms);
        top = mn;
    }
    const float m = wave_max(top), ms = m == kNone ? 0.f : m;
    sum *= __builtin_amdgcn_exp2f(top - ms);
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
#pragma unroll
    for (int i = 0; i < NR; ++i) acc[i] = 0.f;
    for (int s0 = wave; s0 < cnt; s0 += 8 * kWaves) {
        if (s0 != wave) load(s0);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (s0 + e * kWaves < cnt) {
                const float x = __builtin_amdgcn_exp2f(w[e] - ms);
#pragma unroll
                for (int i = 0; i < NR; ++i) acc[i] += x * t[e][i];
            }
    }
#pragma unroll
    for (int i = 0; i < NR; ++i) lds_a[wave][lane + 64 * i] = acc[i];
    __syncthreads();
    const int dim = threadIdx.x;
    if (dim < D) {
        float x = lds_a[0][dim];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) x += lds_a[w][dim];
        x *= sum == 0.f ? 0.f : 1.f / sum;
        char *to = a.out + ((int64_t)b * a.o_seq + (int64_t)head * a.o_head) * ES;
        if constexpr (ST)
            ((__bf16 *)to)[dim] = (__bf16)x;
        else
            ((float *)to)[dim] = x;
    }
    if (a.lse && threadIdx.x == 0)
        a.lse[blockIdx.x] = sum == 0.f ? kNone : (m + __builtin_amdgcn_logf(sum)) * kLn2;
}

// Rows into the cache: a copy, bound by HBM.  One workgroup per block of 32
// positions and head, so that both sides move whole lines: keys go straight to
// their places, lanes in the order of those; values are turned in LDS.
// Sequence b's rows touch at most rows / 32 + 2 blocks, so its items start at
// starts[b] / 32 + 2 b, which needs no sum over the sequences before it.
// 8 heads of 128 in bf16: 4,096 rows 8.1 us (33.6 MB read and written, 4.1
// TB/s; a row at a time, with scattered stores, 27.8), 16 x 1,000 rows 24.4 (131
// MB, 5.4 TB/s; 91).
template <int ST>
__global__ __launch_bounds__(256) void append_kernel(RowsArgs a, int64_t items) {
    using T = typename std::conditional<ST, uint16_t, uint32_t>::type;
    constexpr int E = ST ? 8 : 4;
    extern __shared__ __align__(16) char lds_rows[];  // the block's values [32][dim + E]
    const int dim = a.dim, pieces = dim / E, ld = dim + E;
    T *rows = (T *)lds_rows;
    const bool marked = a.status[2] != 0;  // some page may take no new rows
    for (int64_t w = blockIdx.x; w < items * a.heads; w += gridDim.x) {
        const int64_t item = w / a.heads;
        const int h = (int)(w % a.heads);
        int64_t b = item, blk = 0, row0 = item, count = 1;  // the sequence's rows
        if (a.starts) {
            auto base = [&](int64_t x) { return ((int64_t)a.starts[x] >> 5) + 2 * x; };
            int64_t lo = 0, hi = a.nseq;  // the last one that starts at or before the item
            while (hi - lo > 1) {
                const int64_t mid = (lo + hi) / 2;
                if (base(mid) <= item)
                    lo = mid;
                else
                    hi = mid;
            }
            b = lo;
            blk = item - base(b);
            row0 = a.starts[b];
            count = a.starts[b + 1] - row0;
        }
        const int64_t end = a.lens[b], first = end - count;  // positions
        const int64_t p0 = ((first >> 5) + blk) * kKvBlock;
        if (blk < 0 || count <= 0 || p0 < 0 || p0 >= end) continue;
        char *const at = block_of(a, (int)b, p0, sizeof(T));
        if (!at) {
            if (p0 >> a.page_shift >= a.width && threadIdx.x == 0)
                atomicOr(&a.status[0], kStatusWidth);
            continue;
        }
        if (marked && end <= a.width << a.page_shift) {
            const int last = a.table[b * a.width + ((end - 1) >> a.page_shift)];
            if ((unsigned)last < (unsigned)a.npages && a.closed[last]) continue;
        }
        // positions t of the block that have a row
        const int64_t from = max(row0 < 0 ? first - row0 : first, p0);
        const int64_t to = min(min(end, first + (a.nrows - row0)), p0 + kKvBlock);
        if (from >= to) continue;
        const int t0 = (int)(from - p0), t1 = (int)(to - p0);
        auto row_of = [&](int t) { return row0 + (p0 + t - first); };
        const T *ks = (const T *)a.k + h * a.k_head, *vs = (const T *)a.v + h * a.v_head;
        char *const kd = at + h * a.head_off, *const vd = kd + a.kv_off;
        __syncthreads();  // (the last block's values have been read)
        for (int x = threadIdx.x; x < kKvBlock * pieces; x += 256) {
            const int t = x / pieces, c = x % pieces;
            if (t >= t0 && t < t1)
                *(u32x4_t *)(rows + t * ld + c * E) =
                    load_piece<ST>((const char *)(vs + row_of(t) * a.v_row), c * E, a.v_vec);
        }
        for (int x = threadIdx.x; x < kKvBlock * pieces; x += 256) {
            const int t = x / 16 / pieces * 16 + x % 16, c = x / 16 % pieces;
            if (t >= t0 && t < t1)
                *(u32x4_t *)(kd + x * 16) =
                    load_piece<ST>((const char *)(ks + row_of(t) * a.k_row), c * E, a.k_vec);
        }
        __syncthreads();
        store_values<ST>(rows, ld, (T *)vd, dim, t0, t1);
    }
}

// The same backwards, a workgroup per position: for looking at a cache, not for
// a decoding loop (4,096 positions of 8 x 128 in bf16 21 us).
template <int ST>
__global__ __launch_bounds__(256) void read_kernel(RowsArgs a) {
    using T = typename std::conditional<ST, uint16_t, uint32_t>::type;
    for (int64_t row = blockIdx.x; row < a.nrows; row += gridDim.x) {
        const int64_t pos = a.first + row;
        const char *at = block_of(a, a.b, pos, sizeof(T));
        for (int x = threadIdx.x; x < a.heads * a.dim; x += 256) {
            const int h = x / a.dim, d = x % a.dim;
            T k = 0, v = 0;
            if (at) {
                k = ((const T *)(at + h * a.head_off))[key_place<ST>(pos % kKvBlock, d, a.dim)];
                v = ((const T *)(at + a.kv_off +
                                 h * a.head_off))[value_place<ST>(pos % kKvBlock, d, a.dim)];
            }
            ((T *)a.k_out)[row * a.heads * a.dim + x] = k;
            ((T *)a.v_out)[row * a.heads * a.dim + x] = v;
        }
    }
}

template <int ST, int D, int NW>
hipError_t launch_items(const AttendArgs &a, int64_t items, hipStream_t st) {
    constexpr int DW = D < join_dims(NW) ? D : join_dims(NW);
    const size_t lds = (size_t)NW * std::min(a.group, 16) * (DW + 4) * sizeof(float);
    hipLaunchKernelGGL((attend_kernel<ST, D, NW>), dim3((uint32_t)(items * a.kv_heads * a.gtiles)),
                       dim3(64 * NW), lds, st, a);
    return hipGetLastError();
}

template <int ST, int D>
hipError_t launch_attend(const AttendArgs &a, int64_t items, int waves, bool join, hipStream_t st) {
    if constexpr (D <= kWideDim) {
        if (waves == 8) return launch_items<ST, D, 8>(a, items, st);
    }
    hipError_t e = launch_items<ST, D, kWaves>(a, items, st);
    if (e != hipSuccess || !join) return e;
    hipLaunchKernelGGL((attend_join_kernel<ST, D>), dim3((uint32_t)a.nseq * (uint32_t)a.heads),
                       dim3(64 * kWaves), 0, st, a);
    return hipGetLastError();
}

template <int ST>
hipError_t launch_attend_dim(const AttendArgs &a, int64_t items, int waves, bool join, int dim,
                             hipStream_t st) {
    switch (dim) {
#define VS_DIM(D) \
    case D:       \
        return launch_attend<ST, D>(a, items, waves, join, st);
        VS_DIM(16) VS_DIM(32) VS_DIM(48) VS_DIM(64) VS_DIM(80) VS_DIM(96) VS_DIM(112) VS_DIM(128)
        VS_DIM(144) VS_DIM(160) VS_DIM(176) VS_DIM(192) VS_DIM(208) VS_DIM(224) VS_DIM(240)
        VS_DIM(256)
#undef VS_DIM
    }
    return hipErrorInvalidValue;
}

}  // namespace
}  // namespace vs

using vs::report;
using vs::report_hip;

extern "C" {

int vs_kv_create(int device, int64_t npages, int64_t page_size, int64_t layers, int64_t kv_heads,
                 int64_t head_dim, int dtype, void *memory, vs_kv **out) {
    if (!out) return report(VS_ERR_INVALID, "null output handle");
    *out = nullptr;
    if (npages <= 0 || layers <= 0 || kv_heads <= 0)
        return report(VS_ERR_INVALID, "npages, layers and kv_heads must be > 0");
    if (dtype != VS_DTYPE_F32 && dtype != VS_DTYPE_BF16)
        return report(VS_ERR_INVALID, "unknown dtype code %d", dtype);
    if (page_size < 32 || page_size > 1024 || (page_size & (page_size - 1)))
        return report(VS_ERR_INVALID, "page_size must be a power of two from 32 to 1024 (got %lld)",
                      (long long)page_size);
    if (head_dim <= 0 || head_dim % 16 || head_dim > 256)
        return report(VS_ERR_UNSUPPORTED, "head_dim must be a multiple of 16 up to 256 (got %lld)",
                      (long long)head_dim);
    if (npages > INT32_MAX || kv_heads > 4096 || layers > (1 << 20))
        return report(VS_ERR_UNSUPPORTED, "more than 2^31 - 1 pages, 4096 heads or 2^20 layers");
    if ((uintptr_t)memory % 16) return report(VS_ERR_INVALID, "memory is not 16-byte aligned");
    const int64_t pb = layers * 2 * kv_heads * page_size * head_dim * vs::kv_elem(dtype);
    if (pb > ((int64_t)1 << 46) / npages)
        return report(VS_ERR_OOM, "%lld pages of %lld bytes", (long long)npages, (long long)pb);
    int rc = vs::check_device(device);
    if (rc) return rc;
    vs::DeviceGuard g(device);
    if (g.err != hipSuccess) return report_hip(g.err, "hipSetDevice");
    vs_kv *kv = new (std::nothrow) vs_kv();
    if (!kv) return report(VS_ERR_OOM, "host allocation");
    kv->device = device;
    kv->npages = npages;
    kv->page_size = page_size;
    kv->layers = layers;
    kv->kv_heads = kv_heads;
    kv->head_dim = head_dim;
    kv->dtype = dtype;
    kv->page_bytes = pb;
    kv->mem = (char *)memory;
    kv->num_cu = vs::cu_count(device);
    void *p = nullptr;
    const size_t marks = vs::kStatusWords * sizeof(int32_t) + (size_t)npages;
    hipError_t e = vs::device_alloc(&p, marks);
    kv->status = (int32_t *)p;
    kv->closed = (uint8_t *)(kv->status + vs::kStatusWords);
    if (e == hipSuccess) e = hipMemset(p, 0, marks);
    if (e == hipSuccess) e = hipStreamSynchronize(nullptr);  // (before any stream's call)
    if (e == hipSuccess && !memory) {
        e = vs::device_alloc(&p, (size_t)(npages * pb));
        if (e == hipSuccess) {
            kv->mem = (char *)p;
            kv->owns_mem = true;
        }
    }
    if (e != hipSuccess) {
        if (kv->status) (void)hipFree(kv->status);
        delete kv;
        return report_hip(e, "cache memory");
    }
    *out = kv;
    return VS_OK;
}

void vs_kv_destroy(vs_kv *kv) {
    if (!kv) return;
    vs::DeviceGuard g(kv->device);
    (void)hipDeviceSynchronize();
    kv->scratch.release();
    if (kv->status) (void)hipFree(kv->status);
    if (kv->owns_mem) (void)hipFree(kv->mem);
    delete kv;
}

int64_t vs_kv_page_bytes(const vs_kv *kv) { return kv ? kv->page_bytes : 0; }
void *vs_kv_memory(const vs_kv *kv) { return kv ? kv->mem : nullptr; }

int vs_kv_attend(vs_kv *kv, const vs_kv_seqs *s, int64_t layer, int64_t heads, const void *q,
                 int64_t q_seq, int64_t q_head, const void *k, int64_t k_seq, int64_t k_head,
                 const void *v, int64_t v_seq, int64_t v_head, void *out, int64_t out_seq,
                 int64_t out_head, float *lse, float scale, int64_t window, int64_t sinks,
                 void *stream) {
    if (!kv) return report(VS_ERR_INVALID, "null handle");
    int rc = vs::check_seqs(kv, s);
    if (rc) return rc;
    if (layer < 0 || layer >= kv->layers)
        return report(VS_ERR_INVALID, "layer %lld out of range [0, %lld)", (long long)layer,
                      (long long)kv->layers);
    if (heads <= 0 || heads % kv->kv_heads)
        return report(VS_ERR_INVALID, "heads (%lld) must be a multiple of kv_heads (%lld)",
                      (long long)heads, (long long)kv->kv_heads);
    if (heads > (1 << 16)) return report(VS_ERR_UNSUPPORTED, "more than 65,536 heads");
    if (!k != !v) return report(VS_ERR_INVALID, "k and v are given together or not at all");
    if (window < 0 || sinks < 0) return report(VS_ERR_INVALID, "negative window or sinks");
    if (!std::isfinite(scale * vs::kLog2e))
        return report(VS_ERR_INVALID, "scale is not finite, or too large for its exponentials' base");
    const int64_t e = vs::kv_elem(kv->dtype);
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) % e || (uintptr_t)lse % 4)
        return report(VS_ERR_INVALID, "a buffer is not aligned to its elements");
    for (int64_t x : {q_seq, q_head, k_seq, k_head, v_seq, v_head, out_seq, out_head})
        if (!vs::stride_ok(x)) return report(VS_ERR_INVALID, "stride %lld", (long long)x);
    if (s->nseq == 0) return VS_OK;
    if (!q || !out) return report(VS_ERR_INVALID, "null q or out");
    vs::DeviceGuard g(kv->device);
    if (g.err != hipSuccess) return report_hip(g.err, "hipSetDevice");
    hipStream_t st = (hipStream_t)stream;

    vs::AttendArgs a = {};
    vs::fill_geometry(kv, layer, a);
    a.table = s->table;
    a.lens = s->lens;
    a.width = s->width;
    a.nseq = (int)s->nseq;
    a.npages = (int)kv->npages;
    a.page_shift = __builtin_ctzll((uint64_t)kv->page_size);
    a.q = (const char *)q;
    a.k = (const char *)k;
    a.v = (const char *)v;
    a.out = (char *)out;
    a.q_seq = q_seq;
    a.q_head = q_head;
    a.k_seq = k_seq;
    a.k_head = k_head;
    a.v_seq = v_seq;
    a.v_head = v_head;
    a.o_seq = out_seq;
    a.o_head = out_head;
    a.lse = lse;
    a.heads = (int)heads;
    a.kv_heads = (int)kv->kv_heads;
    a.group = (int)(heads / kv->kv_heads);
    a.gtiles = (a.group + 15) / 16;
    a.scale2 = scale * vs::kLog2e;
    a.window = (int)std::min<int64_t>(window, INT32_MAX);
    a.sinks = (int)std::min<int64_t>(sinks, INT32_MAX);
    a.q_vec = vs::pieces_ok(q, q_seq, q_head, e);
    a.k_vec = vs::pieces_ok(k, k_seq, k_head, e);

    a.status = kv->status;
    a.closed = kv->closed;
    // Work items: whole ones of so many blocks that two or six workgroups come
    // to a CU, and one per sequence for what is left of it.
    const int64_t per_item = (int64_t)a.kv_heads * a.gtiles;
    auto items_of = [&](int64_t wgs) {
        return std::max<int64_t>(1, (wgs + per_item - 1) / per_item);
    };
    a.most_items = (int)items_of(6 * kv->num_cu);
    a.few_items = (int)items_of(kv->num_cu);
    // the most blocks that a sequence of this table can have
    int64_t most = s->width * (kv->page_size / vs::kKvBlock);
    if (window > 0)
        most = std::min(most, (window + vs::kKvBlock - 1) / vs::kKvBlock + 1 +
                                  (sinks + vs::kKvBlock - 1) / vs::kKvBlock);
    // Short sequences are not split: a workgroup of eight waves, or four where
    // there are workgroups enough, goes through one faster than a second launch
    // joins its parts.  How short, by how many workgroups that leaves (8
    // key-value heads of 128, not split against split: 1 sequence of 500
    // positions 8.8 and 9.5 us, of 1,000 11.4 and 9.6; 16 of 1,000 15 and 19; 64
    // of 1,000 55 and 58, 256 of them 214 and 222; lengths far apart want parts
    // earlier: fp32, 16 sequences of 17 to 1,023 16 and 14).
    const int64_t units = most * (e == 2 ? 1 : 2), wgs = s->nseq * per_item;
    const int waves = wgs >= 2 * kv->num_cu || kv->head_dim > vs::kWideDim ? vs::kWaves : 8;
    const int each = wgs < kv->num_cu / 2 ? 2 : wgs < 2 * kv->num_cu ? 4 : 8;
    // (nor are so many sequences that a launch of their parts, or of the join, is none)
    a.unsplit = most <= vs::kMinBlocks || units <= each * waves ||
                !vs::grid_ok((a.most_items + s->nseq) * per_item, 64 * vs::kWaves) ||
                !vs::grid_ok(s->nseq * heads, 64 * vs::kWaves);
    const bool join = !a.unsplit;
    const int64_t items = a.unsplit ? s->nseq : a.most_items + s->nseq;
    if (!vs::grid_ok(items * per_item, 64 * (join ? vs::kWaves : waves)))
        return report(VS_ERR_UNSUPPORTED, "%lld sequences of %lld heads", (long long)s->nseq,
                      (long long)heads);
    if (join) {
        const size_t slots = (size_t)(items * heads);
        const size_t o_bytes = slots * kv->head_dim * sizeof(float);
        const size_t ml_bytes = slots * sizeof(float2);
        const bool planned = s->nseq > vs::kFindSeqs;
        const size_t f_bytes = (size_t)s->nseq * sizeof(int2);
        void *ws = nullptr;
        rc = kv->scratch.get(
            st, o_bytes + ml_bytes + f_bytes + (planned ? (size_t)(items + 1) * sizeof(int32_t) : 0),
            &ws);
        if (rc) return rc;
        a.part_o = (float *)ws;
        a.part_ml = (float2 *)((char *)ws + o_bytes);
        a.first = (int2 *)((char *)ws + o_bytes + ml_bytes);
        if (planned) {
            a.plan = (int32_t *)(a.first + s->nseq);
            a.items = (int)items;
            hipLaunchKernelGGL(vs::attend_plan_kernel, dim3(1), dim3(vs::kPlan), 0, st, a);
            const hipError_t e_ = hipGetLastError();
            if (e_ != hipSuccess) return report_hip(e_, "attend");
        }
    }
    hipError_t err = kv->dtype == VS_DTYPE_BF16
                         ? vs::launch_attend_dim<1>(a, items, join ? vs::kWaves : waves, join,
                                                    (int)kv->head_dim, st)
                         : vs::launch_attend_dim<0>(a, items, join ? vs::kWaves : waves, join,
                                                    (int)kv->head_dim, st);
    if (err != hipSuccess) return report_hip(err, "attend");
    return VS_OK;
}

int vs_kv_append(vs_kv *kv, const vs_kv_seqs *s, int64_t layer, const void *k, int64_t k_row,
                 int64_t k_head, const void *v, int64_t v_row, int64_t v_head,
                 const int32_t *starts, int64_t nrows, void *stream) {
    if (!kv) return report(VS_ERR_INVALID, "null handle");
    int rc = vs::check_seqs(kv, s);
    if (rc) return rc;
    vs::RowsArgs a = {};
    rc = vs::fill_rows(kv, s, layer, a);
    if (rc) return rc;
    if (nrows < 0 || (!starts && nrows != s->nseq))
        return report(VS_ERR_INVALID, "nrows %lld: without starts, one row per sequence",
                      (long long)nrows);
    for (int64_t x : {k_row, k_head, v_row, v_head})
        if (!vs::stride_ok(x)) return report(VS_ERR_INVALID, "stride %lld", (long long)x);
    if (nrows == 0 || s->nseq == 0) return VS_OK;
    if (!k || !v) return report(VS_ERR_INVALID, "null k or v");
    if (((uintptr_t)k | (uintptr_t)v) % vs::kv_elem(kv->dtype) || (uintptr_t)starts % 4)
        return report(VS_ERR_INVALID, "a buffer is not aligned to its elements");
    vs::DeviceGuard g(kv->device);
    if (g.err != hipSuccess) return report_hip(g.err, "hipSetDevice");
    a.starts = starts;
    a.nrows = nrows;
    a.k = (const char *)k;
    a.v = (const char *)v;
    a.k_row = k_row;
    a.k_head = k_head;
    a.v_row = v_row;
    a.v_head = v_head;
    const int64_t e_bytes = vs::kv_elem(kv->dtype);
    a.k_vec = vs::pieces_ok(k, k_row, k_head, e_bytes);
    a.v_vec = vs::pieces_ok(v, v_row, v_head, e_bytes);
    const int64_t items = starts ? nrows / vs::kKvBlock + 2 * s->nseq + 1 : nrows;
    const dim3 grid((uint32_t)std::min<int64_t>(items * kv->kv_heads, 1 << 20));
    const size_t lds = (size_t)vs::kKvBlock * (kv->head_dim * e_bytes + 16);
    if (kv->dtype == VS_DTYPE_BF16)
        hipLaunchKernelGGL(vs::append_kernel<1>, grid, dim3(256), lds, (hipStream_t)stream, a, items);
    else
        hipLaunchKernelGGL(vs::append_kernel<0>, grid, dim3(256), lds, (hipStream_t)stream, a, items);
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? VS_OK : report_hip(e, "append");
}

int vs_kv_read(vs_kv *kv, const vs_kv_seqs *s, int64_t layer, int64_t b, int64_t first, int64_t n,
               void *k_out, void *v_out, void *stream) {
    if (!kv) return report(VS_ERR_INVALID, "null handle");
    int rc = vs::check_seqs(kv, s);
    if (rc) return rc;
    vs::RowsArgs a = {};
    rc = vs::fill_rows(kv, s, layer, a);
    if (rc) return rc;
    if (b < 0 || b >= s->nseq)
        return report(VS_ERR_INVALID, "sequence %lld out of range [0, %lld)", (long long)b,
                      (long long)s->nseq);
    if (first < 0 || n < 0 || first > INT32_MAX - n)
        return report(VS_ERR_INVALID, "positions [%lld, %lld)", (long long)first,
                      (long long)(first + n));
    if (n == 0) return VS_OK;
    if (!k_out || !v_out) return report(VS_ERR_INVALID, "null k_out or v_out");
    if (((uintptr_t)k_out | (uintptr_t)v_out) % vs::kv_elem(kv->dtype))
        return report(VS_ERR_INVALID, "a buffer is not aligned to its elements");
    vs::DeviceGuard g(kv->device);
    if (g.err != hipSuccess) return report_hip(g.err, "hipSetDevice");
    a.nrows = n;
    a.b = (int)b;
    a.first = (int)first;
    a.k_out = (char *)k_out;
    a.v_out = (char *)v_out;
    const dim3 grid((uint32_t)std::min<int64_t>(n, 65536));
    if (kv->dtype == VS_DTYPE_BF16)
        hipLaunchKernelGGL(vs::read_kernel<1>, grid, dim3(256), 0, (hipStream_t)stream, a);
    else
        hipLaunchKernelGGL(vs::read_kernel<0>, grid, dim3(256), 0, (hipStream_t)stream, a);
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? VS_OK : report_hip(e, "read");
}

}  // extern "C"

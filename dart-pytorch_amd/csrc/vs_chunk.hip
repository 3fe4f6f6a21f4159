// vs_chunk.hip -- attention of many new tokens over the paged key-value cache:
// prompts in chunks, drafted tokens, rows that attend to other sequences' states:
// kernels and entry point.
#include <cmath>

#include "vs_device.h"
#include "vs_rows.h"
#include "vs_wave.h"

namespace vs {
namespace {

constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLog2e = 1.44269504088896340736f;
// Workgroups: tiles of 64, 128 or 256 rows of queries, by four waves of 16 or 32
// rows or eight of 32.
constexpr int kSmallTile = 64, kTile = 128, kLargeTile = 256;
constexpr int kSplitSeqs = 384;               // sequences whose pieces each workgroup finds for itself
constexpr int kMinBlocks = 4;                 // per piece of a tile's blocks, at least
constexpr int kLong = 48;                     // blocks per place from which on there are three pieces to one
                                              // (fp32, 4,096 rows of 8/8 of 128 403 us against 466)
constexpr int kWideDim = 128;                 // bf16 heads up to this size have the larger ones
constexpr float kSlack = 256.f;               // the largest weight that is let stand
constexpr int kJoinRows = 4;                  // rows per workgroup of the join

struct ChunkArgs {
    char *pool;
    int64_t page_bytes, layer_off, kv_off, head_off;  // bytes; kv_off from keys to values
    const int32_t *table, *lens, *starts;
    int64_t width;
    int nseq, npages, page_shift;
    int64_t nrows;
    const char *q;
    char *out;
    int64_t q_row, q_head, o_row, o_head;  // elements
    float *lse;
    int heads, kv_heads, group;  // group: query heads per key-value head
    float scale2;                // |scale| * log2(e)
    uint32_t flip;               // sign bits of an element's word, where scale is below 0
    int causal, window, sinks;
    int q_vec;                   // rows readable in 16-byte pieces
    int tile;                    // rows of queries per workgroup
    int exact;                   // bf16 weights are multiplied with all their bits
    int64_t tiles;               // numbers of tiles, with gaps
    int split;                   // tiles are divided along the length
    int slots;                   // pieces at work at once, per key-value head
    int cost;                    // of a full tile's piece, in blocks
    int spread;                  // pieces per place, at most
    int parts;                   // workgroups of the join per tile and key-value head
    int4 *info;                  // how many tiles; then each one's pieces: the first whole one, how
                                 // many, the rest, how many in use; and its sequence and place there
    float *part_o;               // [piece][kv head][row of the tile][dim]
    float4 *part_ml;             // [piece][kv head][row of the tile] reference, sums of weights as they
                                 // are and as they are multiplied
};

// A value that all lanes have, for the scalar registers.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
    return (int64_t)((uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32 | (uint32_t)uniform((int)x));
}

// The rows of a sequence: [row0, row0 + count) of the batch's, row i at position
// i + shift; `cap` the last position that there is, at most.
struct Seq {
    int64_t row0, shift;
    int count, cap;
};

__device__ __forceinline__ Seq seq_of(const ChunkArgs &a, int b) {
    Seq s;
    const int64_t n = max(a.lens[b], 0), most = a.width << a.page_shift;
    int64_t from = b, to = (int64_t)b + 1;
    if (a.starts) {
        from = a.starts[b];
        to = a.starts[b + 1];
    }
    s.shift = n - to;
    s.cap = (int)min(n, most) - 1;
    s.row0 = min(max(from, (int64_t)0), a.nrows);
    s.count = (int)max(min(to, a.nrows) - s.row0, (int64_t)0);
    return s;
}

// Query rows are (row, query head of the group) pairs, the head counting faster, so
// that a tile's rows share their keys and values whatever the group.
__device__ __forceinline__ int tiles_of(const ChunkArgs &a, const Seq &s) {
    return (int)(((int64_t)s.count * a.group + a.tile - 1) / a.tile);
}

// The last position that row x of sequence s sees; -1: none.
__device__ __forceinline__ int last_of(const ChunkArgs &a, const Seq &s, int64_t x) {
    return a.causal ? (int)max(min(s.row0 + x + s.shift, (int64_t)s.cap), (int64_t)-1) : s.cap;
}

// A tile's number: those of sequence b start at base(b), which needs no sum over
// the sequences before it and leaves a gap of one at most.
__device__ __forceinline__ int64_t tile_base(const ChunkArgs &a, int64_t b) {
    const int64_t from = a.starts ? min(max((int64_t)a.starts[b], (int64_t)0), a.nrows) : b;
    return from * a.group / a.tile + b;
}

// The blocks that a tile attends to: nsb from the start, then from wb0 on.
struct Span {
    int nsb, wb0, total;
};

__device__ __forceinline__ Span span_of(const ChunkArgs &a, int low, int high) {
    Span s = {0, 0, 0};
    if (high < 0) return s;
    const int nb = high / kKvBlock + 1;
    if (a.window > 0 && low >= a.window) {
        s.wb0 = (low - a.window + 1) / kKvBlock;
        s.nsb = min(a.sinks / kKvBlock + (a.sinks % kKvBlock != 0), s.wb0);
    }
    s.total = s.nsb + nb - s.wb0;
    return s;
}

// How many blocks any tile of a sequence has, at most.
__device__ __forceinline__ int most_blocks(const ChunkArgs &a, const Seq &s) {
    const int high = s.count ? last_of(a, s, s.count - 1) : -1;
    if (high < 0) return 0;
    const int nb = high / kKvBlock + 1;
    if (a.window <= 0) return nb;
    const int64_t w = ((int64_t)a.window + a.tile / a.group) / kKvBlock + 3 + a.sinks / kKvBlock;
    return (int)min((int64_t)nb, w);
}

__device__ __forceinline__ int64_t wave_sum64(int64_t x) {
#pragma unroll
    for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
    return x;
}

// Piece `piece` of a divided call: the split-th `per` blocks of tile `tile` of
// sequence b.  All whole pieces come first, then what is left of each tile, so
// that the smaller ones fill the places that come free.
struct Piece {
    int b, tile, split, per;
    int first, whole, rest;  // the tile's pieces: first .. first + whole - 1, and rest (-1: none)
    int number, count;       // of the tile among all, and how many they are
};

__device__ __forceinline__ bool find_piece(const ChunkArgs &a, int piece, int lane, Piece &p) {
    int64_t all = 0, bound = 0, filled = 0;
    int count = 0, widest = 0;
    auto look = [&](int b, int &tiles, int &blocks, bool sum) {
        tiles = blocks = 0;
        if (b >= a.nseq) return;
        const Seq s = seq_of(a, b);
        tiles = tiles_of(a, s);
        blocks = most_blocks(a, s);
        if (!sum) return;
        // (causal tiles grow from the first to the last)
        const int least = min(max(last_of(a, s, 0), 0) / kKvBlock + 1, blocks);
        all += ((int64_t)tiles * (blocks + least) + 1) / 2;
        bound += (int64_t)tiles * blocks;
        count += tiles;
        filled += (int64_t)s.count * a.group;
        widest = max(widest, blocks);
    };
    int t0, n0;  // (all there is to read for up to 64 sequences)
    look(lane, t0, n0, true);
    for (int b = lane + 64; b < a.nseq; b += 64) {
        int t, n;
        look(b, t, n, true);
    }
    all = uniform(wave_sum64(all));
    bound = uniform(wave_sum64(bound));
    p.count = count = (int)wave_sum((uint32_t)count);
    if (count > a.tiles) {  // starts that do not ascend: there is no room for so many
        p.count = 0;
        return false;
    }
    widest = uniform((int)wave_max((float)widest));  // (past 2^24 off by two at most: a piece more)
    // Pieces of such a length that all are at work at once where tiles are few, or
    // so many that they spread.  They cost their start and the join of their rows,
    // a.cost blocks for a full tile of kTile rows: where whole tiles take no more than
    // that longer, there are none.
    const int64_t ideal = all / a.slots;
    // (twice as many of causal tiles that grow from nothing: half of theirs are empty.
    // By 2, 3, 4 and 6 per place: fp32, 4,096 rows of 8/8 of 128 536, 466, 586 and 403 us,
    // of 12/12 of 64 304, 339, 326 and 315; two chunks of 511 among 30 single rows
    // 179, 185, 193 and 214; fp32, 6 prompts of 17 to 1,023 of 12/12 of 64 63, 66, 70 and 72)
    const int each = ideal < kLong || a.spread == 2 ? 2 : 2 * bound <= 3 * all ? a.spread / 2 : a.spread;
    const int target = 2 * count <= a.slots ? a.slots - count : each * a.slots;
    // (by the bound, which the pieces' numbers go by: there are no more than
    // target of them and one of each tile)
    p.per = (int)max((bound + target - 1) / target, (int64_t)kMinBlocks);
    const int64_t undivided = count <= a.slots ? widest : max((int64_t)widest, ideal + widest / 2);
    const int64_t full = uniform(wave_sum64(filled)) * 16 / ((int64_t)max(count, 1) * a.tile);  // 16ths
    if (undivided <= ideal + a.cost / 8 + a.cost * full * a.tile / (16 * kTile)) p.per = max(p.per, widest + 2);
    int wholes = 0;
    for (int b0 = 0; b0 < a.nseq; b0 += 64) {
        int t = t0, n = n0;
        if (b0) look(b0 + lane, t, n, false);
        wholes += (int)wave_sum((uint32_t)(t * (n / p.per)));
    }
    const bool is_rest = piece >= wholes;
    int base = 0, rank = wholes, tbase = 0;
    for (int b0 = 0; b0 < a.nseq; b0 += 64) {
        int t = t0, n = n0;
        if (b0) look(b0 + lane, t, n, false);
        const int whole = n / p.per, rest = n == 0 || n % p.per != 0;
        const int wsum = base + prefix_sum(t * whole), rsum = rank + prefix_sum(t * rest);
        const int tsum = tbase + prefix_sum(t);
        const uint64_t past = __ballot((is_rest ? rsum : wsum) > piece);
        if (past) {
            const int l = __builtin_ctzll(past);
            const int tiles = __builtin_amdgcn_readlane(t, l);
            const int w = __builtin_amdgcn_readlane(whole, l), r = __builtin_amdgcn_readlane(rest, l);
            const int first = __builtin_amdgcn_readlane(wsum, l) - tiles * w;
            const int left = __builtin_amdgcn_readlane(rsum, l) - tiles * r;
            p.b = b0 + l;
            p.tile = is_rest ? piece - left : (piece - first) / w;
            p.split = is_rest ? w : (piece - first) % w;
            p.whole = w;
            p.first = first + p.tile * w;
            p.rest = r ? left + p.tile : -1;
            p.number = __builtin_amdgcn_readlane(tsum, l) - tiles + p.tile;
            return true;
        }
        base = __builtin_amdgcn_readlane(wsum, 63);
        rank = __builtin_amdgcn_readlane(rsum, 63);
        tbase = __builtin_amdgcn_readlane(tsum, 63);
    }
    return false;
}

// The larger of the four lanes that share a column (lanes apart by 16).
__device__ __forceinline__ float column_max(float x) {
    typedef unsigned u32pair __attribute__((ext_vector_type(2)));
    u32pair p = __builtin_amdgcn_permlane16_swap(bits_of(x), bits_of(x), false, false);
    x = fmaxf(float_of(p.x), float_of(p.y));
    p = __builtin_amdgcn_permlane32_swap(bits_of(x), bits_of(x), false, false);
    return fmaxf(float_of(p.x), float_of(p.y));
}

// blocks of 32 positions that are staged together
constexpr int blocks_at_once(int st, int dim, int waves, int cols) { return st && dim <= 128 && waves == 8 ? 2 : 1; }
constexpr int buffer_bytes(int st, int dim, int waves, int cols) {
    return blocks_at_once(st, dim, waves, cols) * 2 * kKvBlock * dim * (st ? 2 : 4);
}

// One tile's pass over its blocks, with the running sums of the softmax.  Query
// rows are (row, head of the group) pairs, so all heads of a key-value head share what
// is staged: a step's blocks go through registers into one of two buffers in LDS, in
// the cache's own layout, while the other one is multiplied.  A wave holds 16 kCols
// query rows as columns; lane (r, g) = (lane & 15, lane >> 4).
//   S^T = K Q^T    A operand: key rows (position r, 16 bytes of dimensions g);
//                  B operand: the queries, column r
//   O^T = V^T P^T  A operand: dimension r, the positions of lane group g;
//                  B operand: P^T, S^T's accumulator as it stands
// bf16, kParts = 1: weights are rounded to bf16, half a step (2^-8 of a weight) at
// most; they are divided by the sum of what they are rounded to, so that they add up to
// 1 and one position alone is answered exactly.  lse goes by their sum before that.
// kParts = 3: a weight is multiplied as the sum of three bf16 values, its 24 bits eight
// at a time, so that answers are those of 32-bit weights, rounded once.  That is for
// calls with few rows per sequence (up to 64 rows times heads of the group on average:
// decoding, drafts), as the attention of one new token has it, because it costs them
// little: 64 x 8 rows over 4,000 positions 184 -> 185 us, 4 x 5 over 900 to 30,000 33.3 ->
// 35.3, 1 x 4 over 1,000 15.6 -> 16.3.  Others are bound by the matrix pipe enough
// to pay (32/8 heads of 128, by one, two and three parts): 8,192 rows 570, 859 and 965 us,
// 4,096 164, - and 239, two chunks of 511 among 30 single rows 186, 204 and 224, window 2,048
// 154, 177 and 207; 16 x 40 to 130 rows over 200 to 4,000, 16/16 of 64, 48, 53 and 61.
// fp32 has fp32 products.
//
// What bounds it: the matrix pipe and, beside it, the vector unit (32 positions of 32
// rows are 32 products of 16 cycles at head size 128, and 16 exponentials with four to
// five other instructions each), which overlap only in part.  8,192 rows of 32/8
// heads of 128 571 us (964 TFLOP/s; a library product of 8,192^3 1,394), 4,096 164 us
// (838); of 64 103 us (667); fp32, 4,096 rows of 12 heads of 64 315 us (82 of 154).  Head
// sizes that are no multiple of 32 fill neither the last pieces of a key row nor the
// waves' shares of a block: 4,096 rows of 16/8 of 144 200 us, of 160 150, of 176 246, of
// 192 172, of 208 299, of 224 203, of 240 345, of 256 227.
// What was gained on the way, 8,192 rows: positions, masks and pages in scalar
// registers 952 -> 818 us; keys and values read ahead of their products 810 -> 695; values
// with their lane groups turned, so that no bank is asked twice 695 -> 673; 256 rows per
// staged block 673 -> 602; no maximum in most steps, block flags and addresses ready in
// the lanes 602 -> 553; the sum of the rounded weights, a product with ones, 553 -> 571
// (by the vector unit 577).
// Tiles: 256 rows by eight waves where they fill the card twice over (a workgroup to a
// CU, two blocks a step; half the staging of 128 rows: 552 against 594 us, without the
// rounded weights' sum), 64 rows where even 128 do not fill it (prompts of 256, 512, 1,024
// and 1,500 rows 17, 23, 38 and 55 us against 20, 28, 41 and 60 by 128) and for fp32 and
// heads past 128, whose accumulators fill the registers (head size 256, 4,096 rows of 16/8
// 226 us; by 128 rows 255), 128 between them.  Steps of two blocks leave four waves too few
// registers (4,096 rows 158 us with one, 171 with two, without that sum).
template <int ST, int D, int NW, int kCols, int kParts>
__global__ __launch_bounds__(64 * NW, !ST && D > 192 ? 1 : kParts == 3 && D <= 128 ? 3 : 2) void chunk_kernel(ChunkArgs args) {
    // (what only the loop's edges need is read from the arguments again: held in the
    // scalar registers it would be moved out of them and back in every step)
    const ChunkArgs &a = args;
    const auto again = [] {
        auto *p = (const __attribute__((address_space(4))) ChunkArgs *)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(p));
        return p;
    };
    constexpr int E = ST ? 8 : 4;
    constexpr int ES = 16 / E;           // element size
    constexpr int NC = (D / E + 3) / 4;  // 16-byte pieces per lane of a key row
    constexpr int ND = D / 16;
    constexpr int SB = blocks_at_once(ST, D, NW, kCols);
    constexpr int BLOCK = kKvBlock * D * ES;         // bytes of a block's keys
    constexpr int LOADS = SB * 2 * BLOCK / 1024;     // of 16 bytes per lane, all waves
    constexpr int MINE = (LOADS + NW - 1) / NW;
    constexpr int kTile = NW * kCols * 16;  // rows of queries
    constexpr float kNone = -__builtin_huge_valf();
    extern __shared__ __align__(16) char lds[];  // two buffers: [block][keys, values]
    __shared__ int flagged[2];                   // the step whose values hold NaNs or infinities
    __shared__ float lds_p[NW][kKvBlock][16];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.x % a.kv_heads;
    const int64_t at = blockIdx.x / a.kv_heads;

    // which rows, which blocks
    Piece pc = {};
    if (a.split) {
        const bool found = find_piece(a, (int)at, lane, pc);
        if (at == 0 && kvh == 0 && threadIdx.x == 0) a.info[0].x = pc.count;
        if (!found) return;
    } else {
        const int64_t number = a.tiles - 1 - at;
        pc.b = (int)last_at_or_below(a.nseq, number, lane, [&](int64_t b) { return tile_base(a, b); });
        pc.tile = (int)(number - tile_base(a, pc.b));
        pc.per = INT32_MAX;
    }
    pc.b = uniform(pc.b);
    pc.tile = uniform(pc.tile);
    pc.split = uniform(pc.split);
    Seq sq = seq_of(a, pc.b);
    sq.row0 = uniform(sq.row0);
    sq.shift = uniform(sq.shift);
    sq.count = uniform(sq.count);
    sq.cap = uniform(sq.cap);
    if (pc.tile < 0 || pc.tile >= tiles_of(a, sq)) return;
    // (rows times heads fit 31 bits with a tile to spare)
    const int x0 = pc.tile * kTile, x1 = min(x0 + kTile, sq.count * a.group);
    const int high = uniform(last_of(a, sq, (x1 - 1) / a.group));
    const int low = uniform(last_of(a, sq, x0 / a.group));
    const Span sp = span_of(a, low, high);
    int pieces = 1, j0 = 0, j1 = sp.total;
    if (a.split) {
        pieces = max((sp.total + pc.per - 1) / pc.per, 1);
        if (pc.split >= pieces) return;
        j0 = pc.split * pc.per;
        j1 = min(j0 + pc.per, sp.total);
        if (pc.split == 0 && kvh == 0 && threadIdx.x == 0) {
            a.info[1 + 2 * pc.number] = make_int4(pc.first, pc.whole, pc.rest, pieces);
            a.info[2 + 2 * pc.number] = make_int4(pc.b, pc.tile, 0, 0);
        }
    }

    // the wave's rows: column c * 16 + r is query row `row[c]` of the sequence
    const int w0 = x0 + wave * (16 * kCols), w1 = min(w0 + 16 * kCols, x1);
    const bool busy = w0 < w1;
    const int wave_high = busy ? uniform(last_of(a, sq, (w1 - 1) / a.group)) : -1;
    const int wave_low = busy ? uniform(last_of(a, sq, w0 / a.group)) : -1;
    int last[kCols], below[kCols];  // sees positions above `below` up to `last`, and the sinks
    u32x4_t qf[kCols][NC];
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
        const int x = w0 + c * 16 + r;
        const bool in = x < w1;
        last[c] = in ? last_of(a, sq, x / a.group) : -1;
        below[c] = a.window > 0 ? last[c] - a.window : -1;
        const char *row = a.q + ((sq.row0 + x / a.group) * a.q_row +
                                 (kvh * a.group + x % a.group) * a.q_head) * ES;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            qf[c][i] = u32x4_t{0, 0, 0, 0};
            if (in && i * 4 + g < D / E) {
                qf[c][i] = load_piece<ST>(row, (i * 4 + g) * E, a.q_vec);
#pragma unroll
                for (int w = 0; w < 4; ++w) qf[c][i][w] ^= a.flip;
            }
        }
    }

    // a column's reference (a score times scale2), whether it has none yet (then past
    // kSlack), the lane's sum of weights, and the column's of weights rounded to bf16
    float ref[kCols], unset[kCols], l[kCols];
    f32x4_t lr[kCols];
    f32x4_t o[kCols][ND];
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
        ref[c] = l[c] = 0.f;
        lr[c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        unset[c] = w0 + c * 16 + r < w1 ? 2.f * kSlack : 0.f;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[c][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    // The blocks in order: 64 at a time, lane i looks the i-th up (where it lies; its
    // first position, a multiple of 32, and below that what masks it needs), and
    // those that are on a page are a bit mask.
    constexpr int kTileWhole = 1;  // every row of the tile sees all of the block
    constexpr int kWaveWhole = 2;  // every row of the wave does
    constexpr int kWaveNone = 4;   // no row of the wave sees any of it
    // no block: past all positions, whose last one is 2^31 - 33 at most (a table has
    // fewer than 2^31 of them, in whole blocks)
    constexpr int kNoBlock = (INT32_MAX & ~(kKvBlock - 1)) + kWaveNone;
    char *const head_base = a.pool + a.layer_off + (int64_t)kvh * a.head_off;
    int chunk = j0 - 64, at_pos = 0;
    uint32_t at_low = 0, at_high = 0;
    uint64_t ready = 0;
    auto whole = [&](int pos, int lo, int hi) {
        return (pos + kKvBlock - 1 <= lo) &
               ((a.window == 0) | (pos > hi - a.window) | (pos + kKvBlock <= a.sinks));
    };
    auto refill = [&]() {  // whether there are any left
        do {
            chunk += 64;
            if (chunk >= j1) return false;
            const auto *a = again();
            const int j = min(chunk + lane, j1 - 1);
            const int pos = (j < sp.nsb ? j : j - sp.nsb + sp.wb0) * kKvBlock;
            const int page = a->table[(int64_t)pc.b * a->width + (pos >> a->page_shift)];
            const uint64_t to = (uint64_t)(a->pool + a->layer_off + (int64_t)kvh * a->head_off +
                                           (int64_t)page * a->page_bytes +
                                           (int64_t)(pos & ((1 << a->page_shift) - 1)) * (D * ES));
            at_low = (uint32_t)to;
            at_high = (uint32_t)(to >> 32);
            at_pos = pos | (whole(pos, low, high) ? kTileWhole : 0) |
                     (whole(pos, wave_low, wave_high) ? kWaveWhole : 0) |
                     (pos > wave_high ? kWaveNone : 0);
            ready = __ballot((chunk + lane < j1) & ((unsigned)page < (unsigned)a->npages));
        } while (!ready);
        return true;
    };
    auto next_block = [&](const char *&kb, int &block) {
        if (!ready && !refill()) return false;
        const int i = __builtin_ctzll(ready);
        ready &= ready - 1;
        block = __builtin_amdgcn_readlane(at_pos, i);
        kb = (const char *)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)at_high, i) << 32 |
                            (uint32_t)__builtin_amdgcn_readlane((int)at_low, i));
        return true;
    };
    struct Step {
        int block[SB];
    };
    auto all_of = [](const Step &s, int flag) {
        int x = s.block[0];
#pragma unroll
        for (int b = 1; b < SB; ++b) x &= s.block[b];
        return (x & flag) != 0;
    };
    auto pos_of = [](const Step &s, int b) { return s.block[b] & ~(kKvBlock - 1); };
    const char *kb[SB];  // the next step's blocks
    auto next_step = [&](Step &s) {
        if (!next_block(kb[0], s.block[0])) return false;
#pragma unroll
        for (int b = 1; b < SB; ++b)
            if (!next_block(kb[b], s.block[b])) {
                kb[b] = kb[0];
                s.block[b] = kNoBlock;
            }
        return true;
    };
    const int tile_below = a.window > 0 ? low - a.window : -1;
    auto hides = [&](int p, int lst, int blw) { return (p > lst) | ((p <= blw) & (p >= a.sinks)); };
    // Kilobyte x of a step's: of which block, keys or values, where in them.  (What
    // does not go by the wave is known here.)
    constexpr int KB = BLOCK / 1024;
    auto kilobyte = [&](int i, int &b, int &kv, int &z) {
        const int x = i * NW + wave;
        b = 2 * KB % NW == 0 ? i * NW / (2 * KB) : x / (2 * KB);
        kv = KB % NW == 0 ? i * NW / KB % 2 : x / KB % 2;
        z = KB % NW == 0 ? i * NW % KB + wave : x % KB;
        return LOADS % NW == 0 || x < LOADS;
    };
    const int64_t kv_off = a.kv_off;
    const uint32_t lane_at = lane * 16;
    u32x4_t stage[MINE];
    auto load_step = [&]() {
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
            int b, kv, z;
            if (!kilobyte(i, b, kv, z)) continue;
            const char *p = kb[0];
#pragma unroll
            for (int k = 1; k < SB; ++k) p = b == k ? kb[k] : p;
            p += (kv ? kv_off : 0) + z * 1024;
            stage[i] = *(const u32x4_t *)(p + lane_at);
        }
    };
    // Positions that no row of the tile sees may hold anything, and 0 times a NaN
    // is one: their values become 0.  So do those that are not finite where some
    // rows see them and others do not; they are added by themselves.
    auto clean_step = [&](const Step &s, int step) {
        bool odd = false;
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
            int b, kv, z;
            if (!kilobyte(i, b, kv, z) || !kv) continue;
            int pos = pos_of(s, 0);
#pragma unroll
            for (int k = 1; k < SB; ++k) pos = b == k ? pos_of(s, k) : pos;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int h = ST ? e / 4 : z / (KB / 2);
                const bool hidden = hides(pos + 16 * h + 4 * (lane & 3) + (e & 3), high, tile_below);
                if constexpr (ST) {
                    const uint32_t mask = e % 2 ? 0xFFFF0000u : 0xFFFFu;
                    const uint32_t inf = e % 2 ? 0x7F800000u : 0x7F80u;
                    const bool bad = (stage[i][e / 2] & inf) == inf;
                    odd |= bad & !hidden;
                    stage[i][e / 2] &= hidden | bad ? ~mask : ~0u;
                } else {
                    const bool bad = (stage[i][e] & 0x7F800000u) == 0x7F800000u;
                    odd |= bad & !hidden;
                    stage[i][e] = hidden | bad ? 0 : stage[i][e];
                }
            }
        }
        if (odd) flagged[step & 1] = step;
    };
    // Values go to LDS with a piece's lane group turned by its dimension, so that
    // lanes that are served together, which read pieces 64 bytes apart, meet all
    // banks (lanes 0 to 3, 12 to 15 and 20 to 27 are, and so on).
    const int k_at = lane * 16, v_at = (lane ^ (-(lane >> 4) & 3)) * 16;
    auto store_step = [&](const Step &s, int step) {
        if (!all_of(s, kTileWhole)) clean_step(s, step);
        char *buf = lds + (step & 1) * (SB * 2 * BLOCK);
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
            int b, kv, z;
            if (!kilobyte(i, b, kv, z)) continue;
            *(u32x4_t *)(buf + (b * 2 + kv) * BLOCK + z * 1024 + (kv ? v_at : k_at)) = stage[i];
        }
    };

    if (threadIdx.x < 2) flagged[threadIdx.x] = -1;
    __syncthreads();
    Step cur;
    bool more = next_step(cur);
    if (more) {
        load_step();
        store_step(cur, 0);
    }
    __syncthreads();
    for (int step = 0; more; ++step) {
        Step nxt;
        more = next_step(nxt);
        if (more) load_step();
        const char *buf = lds + (step & 1) * (SB * 2 * BLOCK);
        const bool clear = all_of(cur, kWaveWhole), none = all_of(cur, kWaveNone);
        if (!none) {  // (nor does a wave without rows)
            // One block's products beside another's softmax: S^T = K Q^T of the second
            // while the first's exponentials are taken, O^T += V^T P^T of the first
            // beside the second's.  Pieces of keys and values are replaced by the next
            // block's as soon as they are multiplied.
            f32x4_t s[SB][2][kCols], w[SB][2][kCols];
            bf16x8_t pb[ST ? SB : 1][kCols], first[kCols];
            u32x4_t kf[2][NC], vf[ND];
            auto load_key = [&](int b, int h, int i) {
                // (a piece past the row's end is read again and zeroed)
                const int piece = D % (4 * E) ? min(i * 4 + g, D / E - 1) : i * 4 + g;
                kf[h][i] = *(const u32x4_t *)(buf + b * 2 * BLOCK + ((h * (D / E) + piece) * 16 + r) * 16);
                if (D % (4 * E) && i == NC - 1 && i * 4 + g >= D / E) kf[h][i] = u32x4_t{0, 0, 0, 0};
            };
            const int v_lane = (r * 4 + (g ^ (-(r >> 2) & 3))) * 16;
            auto load_value = [&](int x, int d) {  // of block x, or of half x of fp32's one
                vf[d] = *(const u32x4_t *)(buf + (ST ? x * 2 : 0) * BLOCK + BLOCK +
                                           (ST ? 0 : x * (BLOCK / 2)) + d * 1024 + v_lane);
            };
            auto keys_queries = [&](int b) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int c = 0; c < kCols; ++c) s[b][h][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < NC; ++i) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int c = 0; c < kCols; ++c) {
                            f32x4_t &t = s[b][h][c];
                            if constexpr (ST) {
                                t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                    __builtin_bit_cast(bf16x8_t, kf[h][i]),
                                    __builtin_bit_cast(bf16x8_t, qf[c][i]), t, 0, 0, 0);
                            } else {
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    t = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                        float_of(kf[h][i][e]), float_of(qf[c][i][e]), t, 0, 0, 0);
                            }
                        }
                        if (b + 1 < SB) load_key(b + 1, h, i);
                    }
                }
            };
            auto mask = [&](int b) {
                if (clear) return;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int p = pos_of(cur, b) + 16 * h + 4 * g + i;
#pragma unroll
                        for (int c = 0; c < kCols; ++c)
                            s[b][h][c][i] = hides(p, last[c], below[c]) ? kNone : s[b][h][c][i];
                    }
            };
            // Weights are exp2 of a score less the column's reference.  That stands
            // until a weight is past kSlack: they may be that much larger than 1, so
            // no maximum is taken and nothing is rescaled in most steps.
            auto weights = [&](int b) {
#pragma unroll
                for (int c = 0; c < kCols; ++c)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            w[b][h][c][i] = __builtin_amdgcn_exp2f(
                                __builtin_fmaf(s[b][h][c][i], a.scale2, -ref[c]));
            };
            auto check = [&](int b) {
#pragma unroll
                for (int c = 0; c < kCols; ++c) {
                    float top = unset[c];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 4; ++i) top = fmaxf(top, w[b][h][c][i]);
                    if (__ballot(top > kSlack)) {
                        top = kNone;
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int i = 0; i < 4; ++i) top = fmaxf(top, s[b][h][c][i]);
                        top = column_max(top) * a.scale2;
                        // (a column that has seen nothing yet has no reference: 0)
                        const bool none = unset[c] > 0.f;
                        const float to = top == kNone ? ref[c] : none ? top : fmaxf(ref[c], top);
                        const float f = to == ref[c] || none ? 1.f : __builtin_amdgcn_exp2f(ref[c] - to);
                        if (top != kNone) unset[c] = 0.f;
                        ref[c] = to;
                        l[c] *= f;
#pragma unroll
                        for (int i = 0; i < 4; ++i) lr[c][i] *= f;
#pragma unroll
                        for (int d = 0; d < ND; ++d)
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[c][d][i] *= f;
                        if (b > 0)  // (not among the sums yet)
#pragma unroll
                            for (int h = 0; h < 2; ++h)
#pragma unroll
                                for (int i = 0; i < 4; ++i) w[b - 1][h][c][i] *= f;
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                w[b][h][c][i] = __builtin_amdgcn_exp2f(
                                    __builtin_fmaf(s[b][h][c][i], a.scale2, -to));
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 4; ++i) l[c] += w[b][h][c][i];
                }
            };
            auto round_weights = [&](int b) {
                if constexpr (ST)
#pragma unroll
                    for (int c = 0; c < kCols; ++c)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int i = 0; i < 4; ++i) pb[b][c][4 * h + i] = (__bf16)w[b][h][c][i];
            };
            auto weigh_values = [&](int b) {
                if constexpr (ST) {
                    // what they are divided by in the end: weights that add up to 1 (a
                    // product with ones, whose rows are all the sum)
                    const __bf16 u = (__bf16)1.f;
                    const bf16x8_t ones = {u, u, u, u, u, u, u, u};
#pragma unroll
                    for (int part = 0; part < kParts; ++part) {
                        if constexpr (kParts == 1)
#pragma unroll
                            for (int c = 0; c < kCols; ++c)
                                lr[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pb[b][c], lr[c], 0, 0, 0);
#pragma unroll
                        for (int d = 0; d < ND; ++d) {
#pragma unroll
                            for (int c = 0; c < kCols; ++c)
                                o[c][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                    __builtin_bit_cast(bf16x8_t, vf[d]), pb[b][c], o[c][d], 0, 0, 0);
                            if (b + 1 < SB) {
                                load_value(b + 1, d);
                                __builtin_amdgcn_sched_barrier(0);
                            }
                        }
                        if (part + 1 < kParts) {  // what is left of the weights
#pragma unroll
                            for (int c = 0; c < kCols; ++c) {
                                if (part == 0) first[c] = pb[b][c];
#pragma unroll
                                for (int h = 0; h < 2; ++h)
#pragma unroll
                                    for (int i = 0; i < 4; ++i)
                                        w[b][h][c][i] -= (float)pb[b][c][4 * h + i];
                            }
                            round_weights(b);
                        }
                    }
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int d = 0; d < ND; ++d) {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
#pragma unroll
                                for (int c = 0; c < kCols; ++c)
                                    o[c][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                        float_of(vf[d][i]), w[b][h][c][i], o[c][d], 0, 0, 0);
                            if (h == 0) load_value(1, d);
                        }
                }
            };
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                load_key(0, 0, i);
                load_key(0, 1, i);
            }
            __builtin_amdgcn_sched_barrier(0);
            keys_queries(0);
            mask(0);
            __builtin_amdgcn_sched_barrier(0);
            weights(0);
            if constexpr (SB == 2) keys_queries(1);
#pragma unroll
            for (int d = 0; d < ND; ++d) load_value(0, d);
            __builtin_amdgcn_sched_barrier(0);
            check(0);
            if constexpr (SB == 2) {
                mask(1);
                __builtin_amdgcn_sched_barrier(0);
                weights(1);
                check(1);
            }
#pragma unroll
            for (int b = 0; b < SB; ++b) round_weights(b);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int b = 0; b < SB; ++b) weigh_values(b);
            __builtin_amdgcn_s_setprio(0);
            if (!all_of(cur, kTileWhole) && flagged[step & 1] == step) {
                // Values that are not finite, seen by some rows and not by others: a
                // position at a time, only where it is seen.
#pragma unroll
                for (int b = 0; b < SB; ++b)
#pragma unroll
                    for (int c = 0; c < kCols; ++c) {
                        lds_wave_sync();
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                lds_p[wave][16 * h + 4 * g + i][r] =
                                    ST ? (float)(kParts == 1 ? pb[ST ? b : 0] : first)[c][4 * h + i] : w[b][h][c][i];
                        lds_wave_sync();
                        const auto *a = again();
                        const int pos = min(pos_of(cur, b), high);  // (none is seen where there is no block)
                        const char *vb = head_base + a->kv_off +
                            (int64_t)a->table[(int64_t)pc.b * a->width + (pos >> a->page_shift)] * a->page_bytes +
                            (int64_t)(pos & ((1 << a->page_shift) - 1) & ~(kKvBlock - 1)) * (D * ES);
#pragma unroll 1
                        for (int t = 0; t < kKvBlock; ++t) {
                            if (hides(pos_of(cur, b) + t, last[c], below[c])) continue;
                            const float w = lds_p[wave][t][r];
#pragma unroll
                            for (int d = 0; d < ND; ++d)
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const int place = value_place<ST>(t, d * 16 + g * 4 + i, D);
                                    uint32_t v;
                                    if constexpr (ST)
                                        v = (uint32_t)((const uint16_t *)vb)[place] << 16;
                                    else
                                        v = ((const uint32_t *)vb)[place];
                                    if ((v & 0x7F800000u) == 0x7F800000u)
                                        o[c][d][i] = __builtin_fmaf(w, float_of(v), o[c][d][i]);
                                }
                        }
                    }
            }
        }
        if (more) store_step(nxt, step + 1);
        cur = nxt;
        __syncthreads();
    }

#pragma unroll
    for (int c = 0; c < kCols; ++c) {
        l[c] += __shfl_xor(l[c], 16);
        l[c] += __shfl_xor(l[c], 32);
        const float divisor = ST && kParts == 1 ? lr[c][0] : l[c];
        const int x = w0 + c * 16 + r;
        if (x >= w1) continue;
        const auto *a = again();
        if (pieces == 1) {
            const int64_t row = sq.row0 + x / a->group;
            const int head = kvh * a->group + (int)(x % a->group);
            const float inv = divisor == 0.f ? 0.f : 1.f / divisor;
            char *to = a->out + (row * a->o_row + head * a->o_head + g * 4) * ES;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (ST)
                        ((__bf16 *)to)[d * 16 + i] = (__bf16)(o[c][d][i] * inv);
                    else
                        ((float *)to)[d * 16 + i] = o[c][d][i] * inv;
                }
            if (a->lse && g == 0)
                a->lse[row * a->heads + head] =
                    l[c] == 0.f ? kNone : (ref[c] + __builtin_amdgcn_logf(l[c])) * kLn2;
        } else {
            const int64_t slot = (at * a->kv_heads + kvh) * kTile + (x - x0);
#pragma unroll
            for (int d = 0; d < ND; ++d)
                *(f32x4_t *)(a->part_o + slot * D + d * 16 + g * 4) = o[c][d];
            if (g == 0) a->part_ml[slot] = make_float4(unset[c] > 0.f ? kNone : ref[c], l[c], divisor, 0.f);
        }
    }
}

// Joins the pieces of a tile: a workgroup per kJoinRows rows at a time, whose waves
// take the pieces in turn, several at once.  Bound by the partial sums' bytes: 4 x 5
// rows of 32 heads in some 100 pieces 8 us, 1,052 rows in 2 to 3 each 36 us (which is
// why tiles are divided only where that saves more).
template <int ST, int D>
__global__ __launch_bounds__(256) void chunk_join_kernel(ChunkArgs a) {
    constexpr int kWaves = 4;
    constexpr int L = D <= 16 ? 4 : D <= 32 ? 8 : D <= 64 ? 16 : D <= 128 ? 32 : 64;  // lanes per row
    constexpr int P = 64 / L;          // pieces per wave at once
    constexpr int LD = L * 4 + 4;
    constexpr float kNone = -__builtin_huge_valf();
    __shared__ __align__(16) float lds_o[kWaves][kJoinRows][LD];
    __shared__ float2 lds_l[kWaves][kJoinRows];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int part0 = blockIdx.x % a.parts;
    const int kvh = blockIdx.x / a.parts % a.kv_heads;
    const int number = blockIdx.x / a.parts / a.kv_heads;
    // (as many as there may be: what is not a tile is not looked at)
    const int4 f = a.info[1 + 2 * number], place = a.info[2 + 2 * number];
    const int cnt = f.w;
    if (number >= a.info[0].x || cnt <= 1) return;
    const int kTile = a.tile, tile = place.y;
    const Seq sq = seq_of(a, place.x);
    for (int part = part0; part < kTile / kJoinRows; part += a.parts) {
        const int x0 = tile * kTile + part * kJoinRows;
        const int rows = min(sq.count * a.group - x0, kJoinRows);
        if (rows <= 0) return;
        auto slot_of = [&](int s, int j) {
            const int piece = s < f.y ? f.x + s : f.z;
            return ((int64_t)piece * a.kv_heads + kvh) * kTile + part * kJoinRows + j;
        };
        float ms[kJoinRows], sum[kJoinRows], sumr[kJoinRows];
        f32x4_t acc[kJoinRows];
#pragma unroll
        for (int j = 0; j < kJoinRows; ++j) {
            ms[j] = kNone;
            sum[j] = sumr[j] = 0.f;
            acc[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
        for (int s = lane; s < cnt; s += 64)
#pragma unroll
            for (int j = 0; j < kJoinRows; ++j)
                ms[j] = fmaxf(ms[j], a.part_ml[slot_of(s, min(j, rows - 1))].x);
#pragma unroll
        for (int j = 0; j < kJoinRows; ++j) {
            ms[j] = wave_max(ms[j]);
            ms[j] = ms[j] == kNone ? 0.f : ms[j];
        }
        const int at = min(lane % L * 4, D - 4);
#pragma unroll 2
        for (int s = wave * P + lane / L; s < cnt; s += kWaves * P) {
#pragma unroll
            for (int j = 0; j < kJoinRows; ++j) {
                const int64_t slot = slot_of(s, min(j, rows - 1));
                const float4 ml = a.part_ml[slot];
                const f32x4_t o = *(const f32x4_t *)(a.part_o + slot * D + at);
                const float w = __builtin_amdgcn_exp2f(ml.x - ms[j]);
                sum[j] = __builtin_fmaf(w, ml.y, sum[j]);
                sumr[j] = __builtin_fmaf(w, ml.z, sumr[j]);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[j][i] = __builtin_fmaf(w, o[i], acc[j][i]);
            }
        }
#pragma unroll
        for (int j = 0; j < kJoinRows; ++j) {
#pragma unroll
            for (int d = L; d < 64; d *= 2) {
                sum[j] += __shfl_xor(sum[j], d);
                sumr[j] += __shfl_xor(sumr[j], d);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[j][i] += __shfl_xor(acc[j][i], d);
            }
            if (lane < L) *(f32x4_t *)&lds_o[wave][j][lane * 4] = acc[j];
            if (lane == 0) lds_l[wave][j] = make_float2(sum[j], sumr[j]);
        }
        __syncthreads();
        // a wave per row
        static_assert(kJoinRows == kWaves, "");
        if (wave < rows) {
            float l = 0.f, lr = 0.f, top = ms[0];
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                l += lds_l[w][wave].x;
                lr += lds_l[w][wave].y;
            }
#pragma unroll
            for (int j = 1; j < kJoinRows; ++j) top = wave == j ? ms[j] : top;
            const int x = x0 + wave;
            const int64_t row = sq.row0 + x / a.group;
            const int head = kvh * a.group + (int)(x % a.group);
            const float inv = lr == 0.f ? 0.f : 1.f / lr;
            for (int d = lane; d < D; d += 64) {
                float y = 0.f;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) y += lds_o[w][wave][d];
                const int64_t to = row * a.o_row + head * a.o_head + d;
                if constexpr (ST)
                    ((__bf16 *)a.out)[to] = (__bf16)(y * inv);
                else
                    ((float *)a.out)[to] = y * inv;
            }
            if (a.lse && lane == 0)
                a.lse[row * a.heads + head] = l == 0.f ? kNone : (top + __builtin_amdgcn_logf(l)) * kLn2;
        }
        __syncthreads();
    }
}

template <int ST, int D, int NW, int C, int P = 1>
hipError_t launch_tiles(const ChunkArgs &a, int64_t wgs, hipStream_t st) {
    constexpr int lds = 2 * buffer_bytes(ST, D, NW, C);
    if constexpr (lds + sizeof(float) * NW * kKvBlock * 16 + 64 > 65536) {
        const hipError_t e = hipFuncSetAttribute((const void *)chunk_kernel<ST, D, NW, C, P>,
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((chunk_kernel<ST, D, NW, C, P>), dim3((uint32_t)wgs), dim3(64 * NW), lds, st, a);
    return hipGetLastError();
}

template <int ST, int D>
hipError_t launch_chunk(const ChunkArgs &a, int64_t wgs, hipStream_t st) {
    hipError_t e = hipSuccess;
    if constexpr (ST && D <= kWideDim) {
        if (a.tile == kLargeTile) return launch_tiles<ST, D, 8, 2>(a, wgs, st);
        if (a.tile == kTile) e = launch_tiles<ST, D, 4, 2>(a, wgs, st);
    }
    if (a.tile == kSmallTile)
        e = ST && a.exact ? launch_tiles<ST, D, 4, 1, ST ? 3 : 1>(a, wgs, st) : launch_tiles<ST, D, 4, 1>(a, wgs, st);
    if (e != hipSuccess || !a.split) return e;
    hipLaunchKernelGGL((chunk_join_kernel<ST, D>),
                       dim3((uint32_t)(a.tiles * a.kv_heads * a.parts)), dim3(256), 0, st, a);
    return hipGetLastError();
}

template <int ST>
hipError_t launch_chunk_dim(const ChunkArgs &a, int64_t wgs, int dim, hipStream_t st) {
    switch (dim) {
#define VS_DIM(D) \
    case D:       \
        return launch_chunk<ST, D>(a, wgs, st);
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

int vs_kv_attend_rows(vs_kv *kv, const vs_kv_seqs *s, int64_t layer, int64_t heads, const void *q,
                      int64_t q_row, int64_t q_head, void *out, int64_t out_row, int64_t out_head,
                      float *lse, const int32_t *starts, int64_t nrows, float scale, int causal,
                      int64_t window, int64_t sinks, void *stream) {
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
    if (nrows < 0 || (!starts && nrows != s->nseq))
        return report(VS_ERR_INVALID, "nrows %lld: without starts, one row per sequence",
                      (long long)nrows);
    if (window < 0 || sinks < 0) return report(VS_ERR_INVALID, "negative window or sinks");
    if (window > 0 && !causal)
        return report(VS_ERR_INVALID, "a window is of causal rows");
    if (!std::isfinite(scale * vs::kLog2e))
        return report(VS_ERR_INVALID, "scale is not finite, or too large for its exponentials' base");
    const int64_t e = vs::kv_elem(kv->dtype), group = heads / kv->kv_heads;
    if (((uintptr_t)q | (uintptr_t)out) % e || ((uintptr_t)lse | (uintptr_t)starts) % 4)
        return report(VS_ERR_INVALID, "a buffer is not aligned to its elements");
    for (int64_t x : {q_row, q_head, out_row, out_head})
        if (!vs::stride_ok(x, nrows)) return report(VS_ERR_INVALID, "stride %lld", (long long)x);
    if (s->nseq == 0 || nrows == 0) return VS_OK;
    if (!q || !out) return report(VS_ERR_INVALID, "null q or out");
    if (nrows > (INT32_MAX - 1024) / group)
        return report(VS_ERR_UNSUPPORTED, "%lld rows of %lld heads", (long long)nrows, (long long)heads);
    // Rows are answered while others are read.
    const vs::Extent from(q, q_row, q_head, nrows, heads, kv->head_dim, e),
        to(out, out_row, out_head, nrows, heads, kv->head_dim, e);
    const bool same = q == out && (q_row == out_row || nrows == 1) && (q_head == out_head || heads == 1);
    if (!same && vs::meet(from, to))
        return report(VS_ERR_INVALID, "out overlaps q (in place, it is q with its strides)");
    if (vs::overlap(lse, nrows * heads * 4, to.low, to.bytes) ||
        vs::overlap(lse, nrows * heads * 4, from.low, from.bytes))
        return report(VS_ERR_INVALID, "lse overlaps q or out");
    if (vs::over_places(to, s, starts) ||
        (lse && vs::over_places(vs::Extent(lse, 0, 0, 1, 1, nrows * heads, 4), s, starts)))
        return report(VS_ERR_INVALID, "out or lse overlaps starts, lens or table");
    vs::DeviceGuard g(kv->device);
    if (g.err != hipSuccess) return report_hip(g.err, "hipSetDevice");
    hipStream_t st = (hipStream_t)stream;

    vs::ChunkArgs a = {};
    vs::fill_geometry(kv, layer, a);
    a.table = s->table;
    a.lens = s->lens;
    a.starts = starts;
    a.width = s->width;
    a.nseq = (int)s->nseq;
    a.npages = (int)kv->npages;
    a.page_shift = __builtin_ctzll((uint64_t)kv->page_size);
    a.nrows = nrows;
    a.q = (const char *)q;
    a.out = (char *)out;
    a.q_row = q_row;
    a.q_head = q_head;
    a.o_row = out_row;
    a.o_head = out_head;
    a.lse = lse;
    a.heads = (int)heads;
    a.kv_heads = (int)kv->kv_heads;
    a.group = (int)group;
    // A reference is the largest product times the scale, so that is above 0 (0
    // itself as so little that nothing of it is left).
    a.scale2 = std::max(std::fabs(scale * vs::kLog2e), 0x1p-126f);
    a.flip = scale < 0 ? (e == 2 ? 0x80008000u : 0x80000000u) : 0;
    a.causal = causal != 0;
    a.window = (int)std::min<int64_t>(window, INT32_MAX);
    a.sinks = (int)std::min<int64_t>(sinks, INT32_MAX - 64);
    a.q_vec = vs::pieces_ok(q, q_row, q_head, e);
    const int64_t most = s->width * (kv->page_size / vs::kKvBlock);
    // Which tile: see the kernel.  Few rows per sequence never fill a larger one; and
    // prompts (the table has no more than four times their rows) have tiles that grow
    // from the first to the last, which small ones spread: 32/8 heads of 128, 512 rows
    // over 512, 1,500 and 8,192 positions 23, 43 and 171 us by 64, 28, 53 and 122 by 128
    // (1,000 over 5,000 139 and 146: the limit is on the safe side there).
    auto tiles_of = [&](int tile) { return nrows * group / tile + s->nseq; };
    a.tile = vs::kSmallTile;
    const bool few = nrows * group <= s->nseq * vs::kSmallTile;  // per sequence
    const bool prompts = tiles_of(vs::kSmallTile) * a.kv_heads <= 4 * kv->num_cu &&
                         most * vs::kKvBlock * s->nseq <= 4 * nrows;
    if (e == 2 && kv->head_dim <= vs::kWideDim && !few && !prompts)
        a.tile = tiles_of(vs::kLargeTile) * a.kv_heads >= 4 * kv->num_cu ? vs::kLargeTile : vs::kTile;
    a.exact = few;  // (the weights' bits: see the kernel)
    a.tiles = tiles_of(a.tile);
    a.split = a.tiles * a.kv_heads < 4 * kv->num_cu && s->nseq <= vs::kSplitSeqs && most > 4;
    int64_t wgs = a.tiles * a.kv_heads;
    if (a.split) {
        a.slots = (int)std::max<int64_t>(1, 2 * kv->num_cu / a.kv_heads);
        // What pieces cost, in blocks (a tile's start and join take about as long as so
        // many; fp32's blocks take longer).  bf16, 32/8 heads of 128, by 16, 32, 48, 64 and
        // 96: 1,500 rows 64, 64, 55, 55 and 55 us, 3,000 196, 196, 142, 142 and 142, 512 over
        // 2,500 62, 62, 62, 79 and 80.  fp32, 12/12 of 64, by 0, 16, 32 and 48: 512 rows 28, 28,
        // 33 and 33, 6 prompts of 17 to 1,023 63, 63, 63 and 58.
        a.cost = e == 2 ? 48 : 16;
        // (so many workgroups that those without work are soon through)
        a.parts = (int)std::clamp<int64_t>(4096 / (a.tiles * a.kv_heads), 1, a.tile / vs::kJoinRows);
        a.spread = a.tiles * most < vs::kLong * a.slots ? 2 : 6;
        const int64_t pieces = a.spread * a.slots + a.tiles, slots = pieces * a.kv_heads * a.tile;
        const size_t o_bytes = (size_t)slots * kv->head_dim * sizeof(float);
        const size_t ml_bytes = (size_t)slots * sizeof(float4);
        void *ws = nullptr;
        rc = kv->scratch.get(st, o_bytes + ml_bytes + (size_t)(2 * a.tiles + 1) * sizeof(int4), &ws);
        if (rc) return rc;
        a.part_o = (float *)ws;
        a.info = (int4 *)((char *)ws + o_bytes + ml_bytes);
        a.part_ml = (float4 *)((char *)ws + o_bytes);
        wgs = pieces * a.kv_heads;
    }
    if (!vs::grid_ok(wgs, a.tile == vs::kLargeTile ? 512 : 256))
        return report(VS_ERR_UNSUPPORTED, "%lld rows of %lld heads", (long long)nrows, (long long)heads);
    const hipError_t err = kv->dtype == VS_DTYPE_BF16
                               ? vs::launch_chunk_dim<1>(a, wgs, (int)kv->head_dim, st)
                               : vs::launch_chunk_dim<0>(a, wgs, (int)kv->head_dim, st);
    return err == hipSuccess ? VS_OK : report_hip(err, "attend");
}

}  // extern "C"

// vs_beam.hip -- beam search: the choice of the next beams over beams and
// vocabulary, and the reordering of their states.
#include "vs_logits.h"

namespace vs {
namespace {

constexpr int kMaxBeams = 128;
constexpr int kMostSteps = 64;      // per piece
constexpr int kMergeCap = 1024;
constexpr int kMergeThreads = 512;
constexpr int kManyK = 16;          // past it, thresholds come from more than one wave's lanes
constexpr int kWide = 16;           // entries per thread that a merge holds in registers

struct BeamArgs {
    const char *logits;
    int64_t row_stride;  // elements
    int64_t vocab;
    int nreq, nbeam, k, npieces, steps;  // pieces per row, steps per piece
    const float *scores;
    const uint8_t *finished;
    int64_t eos;
    float *scores_out;
    int32_t *tokens_out, *parents_out;
    uint8_t *finished_out;
    float2 *stat;        // [row][piece] maximum and sum of exp(x - maximum)
    float *top_v;        // [row][piece][k] the piece's k largest logits, best first
    int32_t *top_t;      // their tokens; -inf and -1 where there are fewer
};

// One pass over the logits.  A wave takes a piece of a row (every fourth step
// of a stretch that the workgroup's waves read together), 64 PER logits at a
// time, and leaves the piece's maximum and exponential sum (for the row's log
// sum exp) and its k largest logits.
// The list in LDS takes what is at or above a threshold that k logits seen so
// far reach: the k-th largest of the lanes' running maxima, found by bisection
// on ballots.  In most steps of a piece as short as a call's are something is,
// so large calls take steps of twice the length: half the searches.
// Large batches in fp32 are bound by HBM: 64 x 8 x 128,000, k = 8, some beams
// ended, 46 us (232 MB read: 5.0 TB/s).  bf16 has half the bytes for the same
// work and is bound by that, 32 us.  1 x 4 x 50,001 takes 4.9 us, latency.
// Long steps are held to six waves a SIMD, for which bf16 spills two
// registers; with five and none spilled 38.2 against 37.4 us with the merge at 64 x
// 8 x 128,000, k = 8, 56.8 against 55.8 at 128 x 16 x 30,000, k = 32.
template <int ST, int PER>
__global__ __launch_bounds__(256, PER == kLongStep ? 6 : 1) void beam_piece_kernel(BeamArgs a) {
    using S = Step<ST, PER>;
    constexpr int kStep = 64 * PER;
    __shared__ uint64_t lists[4][kCap];
    __shared__ uint32_t maxima[256];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint64_t *cand = lists[wave];
    const uint32_t slot = blockIdx.x * 4 + wave;
    if (slot >= (uint32_t)(a.nreq * a.nbeam) * (uint32_t)a.npieces) return;
    const uint32_t row = slot / (uint32_t)a.npieces;
    // a beam without continuations of its own: its logits do not matter
    if (!(a.scores[row] > VS_NINF) || (a.finished && a.finished[row])) return;
    const char *base = a.logits + row * a.row_stride * S::ES;
    const int vocab = (int)a.vocab;
    // four waves share a stretch of the row and take its steps in turn
    const int share = (int)(slot % (uint32_t)a.npieces) >> 2;
    const int begin = (share * 4 * a.steps + wave) * kStep;
    const int end = min((share + 1) * 4 * a.steps * kStep, vocab);
    constexpr int kNext = 4 * kStep;

    float run = VS_NINF;    // the lane's maximum so far
    float top = VS_NINF;    // the wave's
    float sum = 0.f;        // of exp(x - top), the lane's share
    float thr = -__FLT_MAX__;  // (so -inf is no candidate)
    int n = 0;
    // With many candidates the first threshold is found over the four waves'
    // first steps together, which leaves each a quarter of them (k = 32, 128 x 16
    // x 30,000 bf16 46 against 36 us, k = 24, 50 x 12 x 50,000 with the merge 46
    // against 42.5; k = 16 the same; k = 8 and 10 a us longer for the barrier).
    const bool together = PER == kLongStep && a.k > kManyK;
    S step;
    step.load(base, begin, vocab, lane);  // (past the row's end: nothing but -inf)
    for (int first = begin;;) {
        const S x = step;
        // (a short step's next one is in flight meanwhile; beside a long one are
        // other waves', and registers for more of those are worth more: 28.1
        // against 26.8 us at 97 x 5 x 49,096)
        if (PER == kShortStep && first + kNext < end) step.load(base, first + kNext, vocab, lane);
        float most = fmaxf(x.value(0), x.value(1));
#pragma unroll
        for (int i = 2; i < PER; i += 2) most = max3(most, x.value(i), x.value(i + 1));
        if (__ballot(most > top)) {
            const float w = wave_max(most);
            sum *= __builtin_amdgcn_exp2f((top - w) * kLog2e);  // (0 at first: top is -inf)
            top = w;
        }
        if (together && first == begin) {
            // (all waves of the workgroup are here: they share a row)
            maxima[threadIdx.x] = code_of(most);
            __syncthreads();
            uint32_t code[4], high = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                code[j] = maxima[lane + 64 * j];
                high = max(high, code[j]);
            }
            high = code_of(wave_max(value_of(high)));
            const uint32_t low = code_of(thr), apart = low ^ max(low, high);
            uint32_t bit = apart ? 0x80000000u >> __builtin_clz(apart) : 0;
            uint32_t t = low & ~(2 * bit - (bit != 0));
            for (; bit > (ST ? 0x8000u : 0u); bit >>= 1) {  // (bf16: 16 bits tell)
                int cnt = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) cnt += __popcll(__ballot(code[j] >= (t | bit)));
                if (cnt >= a.k) {
                    t |= bit;
                    if (cnt == a.k) break;
                }
            }
            if (t > low) thr = value_of(t);
        }
        if (__ballot(most >= thr)) {
            run = fmaxf(run, most);
            if (!together || first != begin) {
                // the k-th largest of the lanes' maxima: no lower than the last
                // one, whose leading bits that the largest has too are its
                const uint32_t code = code_of(run), low = code_of(thr);
                const uint32_t apart = low ^ max(low, code_of(top));
                uint32_t bit = apart ? 0x80000000u >> __builtin_clz(apart) : 0;
                uint32_t t = low & ~(2 * bit - (bit != 0));
                for (; bit > (ST ? 0x8000u : 0u); bit >>= 1) {  // (bf16: 16 bits tell)
                    const int cnt = __popcll(__ballot(code >= (t | bit)));
                    if (cnt >= a.k) {
                        t |= bit;
                        if (cnt == a.k) break;
                    }
                }
                if (t > code_of(thr)) thr = value_of(t);
            }
            const int n0 = n;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const float v = x.value(i);
                const uint64_t in = __ballot(v >= thr);
                if (in) {
                    const int at = n + below(in);
                    if (v >= thr && at < kCap) cand[at] = key_of(v, S::token(first, i, lane));
                    n += __popcll(in);
                }
            }
            if (n > kCap) {
                // more than the list holds, ties mostly: again, a register at a
                // time, cut to the k best in between.  What ties with the k-th
                // of these in a later step has a higher token and is out.
                n = n0;
#pragma unroll 1
                for (int i = 0; i < PER; ++i) {
                    const float v = S::reload(base, first, i, vocab, lane);
                    const uint64_t in = __ballot(v >= thr);
                    if (!in) continue;
                    if (n > kCap - 64) {
                        cut_list(cand, n, a.k, lane);
                        n = min(n, a.k);
                    }
                    if (v >= thr) cand[n + below(in)] = key_of(v, S::token(first, i, lane));
                    n += __popcll(in);
                }
                lds_wave_sync();
                if (n >= a.k) {
                    cut_list(cand, n, a.k, lane);
                    n = a.k;
                    thr = value_of((uint32_t)(cand[a.k - 1] >> 32) + 1);
                }
            }
        }
        const float ref = top == VS_NINF ? 0.f : top;
#pragma unroll
        for (int i = 0; i < PER; ++i) sum += __builtin_amdgcn_exp2f((x.value(i) - ref) * kLog2e);
        if (PER != kShortStep && first + kNext < end) step.load(base, first + kNext, vocab, lane);
        first += kNext;
        if (first >= end) break;
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if (lane == 0) a.stat[slot] = make_float2(top, sum);
    float *ov = a.top_v + (int64_t)slot * a.k;
    int32_t *ot = a.top_t + (int64_t)slot * a.k;
    lds_wave_sync();
    for (int c = lane; c < n; c += 64) {
        const uint64_t me = cand[c];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) rank += cand[j] > me;
        if (rank < a.k) {
            ov[rank] = value_of((uint32_t)(me >> 32));
            ot[rank] = (int)~(uint32_t)me;
        }
    }
    for (int c = n + lane; c < a.k; c += 64) {
        ov[c] = VS_NINF;
        ot[c] = -1;
    }
}

struct Cand {
    double total;
    float v;
    int beam, token;
};

__device__ __forceinline__ bool better(const Cand &a, const Cand &b) {
    if (a.total != b.total) return a.total > b.total;
    if (a.beam != b.beam) return a.beam < b.beam;
    if (a.v != b.v) return a.v > b.v;
    return a.token < b.token;
}

// One workgroup per request: the rows' log sum exp from the pieces, then the
// k best of the pieces' candidates, in 64 bits.  What bounds it is the chain
// of loads that wait for each other, so there are two: the pieces' statistics
// with their lists' first entries, and then, at once, all entries of the lists
// whose first is at or above a threshold that k first entries reach (k lists,
// ties aside).  1 x 4 x 50,001, k = 4 4.4 to 5 us; 64 x 8 x 128,000,
// k = 8 5.7 to 6.7 us.
__global__ __launch_bounds__(kMergeThreads) void beam_merge_kernel(BeamArgs a) {
    // total = (logit - largest) + (score - log of the sum of exponentials): in
    // this order no size of the logits costs the total its digits
    __shared__ double offset[kMaxBeams];  // score - log sum; NaN: no candidates
    __shared__ float largest[kMaxBeams];
    __shared__ double own[kMaxBeams];     // a finished beam's score; NaN: not finished, or no eos
    __shared__ float best[kMergeThreads];
    __shared__ Cand list[kMergeCap];
    __shared__ int picked[kMergeCap];     // lists to read whole
    __shared__ int place[kMergeCap];
    __shared__ int nlist, npicked;
    __shared__ int counts[2][kMergeThreads / 64];
    __shared__ float thr;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = blockIdx.x;
    const int64_t row0 = (int64_t)r * a.nbeam;
    const double none = -__builtin_huge_val();
    const int lists = a.nbeam * a.npieces;
    // a thread's first entries, in flight while the statistics are summed
    constexpr int kHeads = 2;
    float head[kHeads];
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
        const int i = threadIdx.x + j * kMergeThreads;
        head[j] = i < lists ? a.top_v[(row0 * a.npieces + i) * a.k] : VS_NINF;
    }
    if (threadIdx.x == 0) nlist = npicked = 0;
    for (int w = wave; w < a.nbeam; w += kMergeThreads / 64) {
        // (loaded whether the beam is alive or not: what is not needed is not used)
        const int64_t row = row0 + w;
        const float score = a.scores[row];
        const float2 *st = a.stat + row * a.npieces;
        const float2 x = lane < a.npieces ? st[lane] : make_float2(VS_NINF, 0.f);
        const bool ended = a.finished && a.finished[row];
        const bool alive = score > VS_NINF;
        double off = __builtin_nan("");
        if (alive && !ended) {
            float top = x.x;
            for (int p = 64 + lane; p < a.npieces; p += 64) top = fmaxf(top, st[p].x);
#pragma unroll
            for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
            const float ref = top == VS_NINF ? 0.f : top;
            double sum = (double)(x.y * __builtin_amdgcn_exp2f((x.x - ref) * kLog2e));
            for (int p = 64 + lane; p < a.npieces; p += 64)
                sum += (double)(st[p].y * __builtin_amdgcn_exp2f((st[p].x - ref) * kLog2e));
#pragma unroll
            for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
            // (a NaN or +inf among the logits makes the sum a NaN; nothing but -inf makes it 0)
            if (sum > 0.0) off = (double)score - log(sum);
            if (lane == 0) largest[w] = top;
        }
        if (lane == 0) {
            offset[w] = off;
            own[w] = alive && ended && a.eos >= 0 && a.eos < a.vocab ? (double)score
                                                                     : __builtin_nan("");
        }
    }
    __syncthreads();

    // the total of logit v of list i; NaN where there is none
    auto total_of = [&](int i, float v) {
        const int w = i / a.npieces;
        return v > VS_NINF ? offset[w] + ((double)v - (double)largest[w]) : __builtin_nan("");
    };
    double mine = none;
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
        const int i = threadIdx.x + j * kMergeThreads;
        if (i < lists) mine = fmax(mine, total_of(i, head[j]));  // (fmax passes NaNs over)
    }
    for (int i = threadIdx.x + kHeads * kMergeThreads; i < lists; i += kMergeThreads)
        mine = fmax(mine, total_of(i, a.top_v[(row0 * a.npieces + i) * a.k]));
    if ((int)threadIdx.x < a.nbeam) mine = fmax(mine, own[threadIdx.x]);
    // The threshold is compared in 32 bits: rounding keeps the order, so what
    // is among the k best is at or above it there too.
    best[threadIdx.x] = (float)mine;
    __syncthreads();
    if (wave == 0) {
        uint32_t t = 0;
        if (a.k <= kManyK) {
            float m = best[lane];
#pragma unroll
            for (int j = 1; j < kMergeThreads / 64; ++j) m = fmaxf(m, best[lane + 64 * j]);
            const uint32_t code = code_of(m);
            for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
                const int cnt = __popcll(__ballot(code >= (t | bit)));
                if (cnt >= a.k) {
                    t |= bit;
                    if (cnt == a.k) break;
                }
            }
        } else {
            // (of 64 maxima the k-th largest would be a weak threshold: 20 x 64 x
            // 50,000, k = 64, with what follows below 434 against 168 us)
            uint32_t code[kMergeThreads / 64];
#pragma unroll
            for (int j = 0; j < kMergeThreads / 64; ++j) code[j] = code_of(best[lane + 64 * j]);
            for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
                int cnt = 0;
#pragma unroll
                for (int j = 0; j < kMergeThreads / 64; ++j)
                    cnt += __popcll(__ballot(code[j] >= (t | bit)));
                if (cnt >= a.k) {
                    t |= bit;
                    if (cnt == a.k) break;
                }
            }
        }
        // (a code below -inf's: all lanes count, and so does everything)
        if (lane == 0) thr = t < code_of(VS_NINF) ? VS_NINF : value_of(t);
    }
    __syncthreads();
    const float t = thr;
    auto pick = [&](int i, double total) {
        if (!((float)total >= t)) return;
        const int at = atomicAdd(&npicked, 1);
        if (at < kMergeCap) picked[at] = i;
    };
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
        const int i = threadIdx.x + j * kMergeThreads;
        if (i < lists) pick(i, total_of(i, head[j]));
    }
    for (int i = threadIdx.x + kHeads * kMergeThreads; i < lists; i += kMergeThreads)
        pick(i, total_of(i, a.top_v[(row0 * a.npieces + i) * a.k]));
    __syncthreads();
    const int lots = npicked;
    // what is at or above `low`: of the picked lists, and of the finished beams
    auto gather = [&](float low) {
        auto add = [&](const Cand &c) {
            const int at = atomicAdd(&nlist, 1);
            if (at < kMergeCap) list[at] = c;
        };
        if ((int)threadIdx.x < a.nbeam && (float)own[threadIdx.x] >= low)
            add({own[threadIdx.x], 0.f, (int)threadIdx.x, (int)a.eos});
        if (lots <= kMergeCap) {
            for (int x = threadIdx.x; x < lots * a.k; x += kMergeThreads) {
                const int i = picked[x / a.k];
                const int64_t at = (row0 * a.npieces + i) * a.k + x % a.k;
                const float v = a.top_v[at];
                const int token = a.top_t[at];
                const double total = total_of(i, v);
                if ((float)total >= low) add({total, v, i / a.npieces, token});
            }
        }
        __syncthreads();
        return nlist;
    };
    int n = gather(t);
    if (n > kMergeCap && lots <= kMergeCap) {
        // More than there is room for (the beams' scores lie far apart, and one
        // beam's lists outdo the others' first entries): the k-th largest of the
        // lists' entries, or as many first ones as fit the registers, by
        // counting over the workgroup.
        uint32_t code[kWide];
        const int deep = min(a.k, kWide * kMergeThreads / lots), most = lots * deep;
#pragma unroll
        for (int j = 0; j < kWide; ++j) {
            const int x = threadIdx.x + j * kMergeThreads;
            code[j] = 0;
            if (x < most) {
                const int i = picked[x / deep];
                const double total =
                    total_of(i, a.top_v[(row0 * a.npieces + i) * a.k + x % deep]);
                if (total == total) code[j] = code_of((float)total);
            }
        }
        uint32_t c = 0;
        int flip = 0;
        for (uint32_t bit = 0x80000000u; bit; bit >>= 1, flip ^= 1) {
            int cnt = 0;
#pragma unroll
            for (int j = 0; j < kWide; ++j)
                if (j * kMergeThreads < most)
                    cnt += __popcll(__ballot(code[j] >= (c | bit)));
            if (lane == 0) counts[flip][wave] = cnt;
            __syncthreads();
            cnt = 0;
#pragma unroll
            for (int w = 0; w < kMergeThreads / 64; ++w) cnt += counts[flip][w];
            if (cnt >= a.k) {
                c |= bit;
                if (cnt == a.k) break;
            }
        }
        if (threadIdx.x == 0) nlist = 0;
        __syncthreads();
        n = gather(fmaxf(t, c < code_of(VS_NINF) ? VS_NINF : value_of(c)));
    }
    const int64_t o0 = (int64_t)r * a.k;
    auto put = [&](int s, const Cand &c) {
        a.scores_out[o0 + s] = (float)c.total;
        a.tokens_out[o0 + s] = c.token;
        a.parents_out[o0 + s] = (int32_t)(row0 + c.beam);
        if (a.finished_out) a.finished_out[o0 + s] = c.token == a.eos;
    };
    auto put_none = [&](int s) {
        a.scores_out[o0 + s] = VS_NINF;
        a.tokens_out[o0 + s] = -1;
        a.parents_out[o0 + s] = -1;
        if (a.finished_out) a.finished_out[o0 + s] = 0;
    };
    if (lots <= kMergeCap && n <= kMergeCap) {
        // Many more than k (few lists, or many of them finished, make the first
        // entries a weak threshold): the k-th largest of them all, as above.
        float t2 = t;
        if (n > 4 * a.k) {
            if (wave == 0) {
                uint32_t code[kMergeCap / 64];
#pragma unroll
                for (int j = 0; j < kMergeCap / 64; ++j)
                    code[j] = lane + 64 * j < n ? code_of((float)list[lane + 64 * j].total) : 0;
                uint32_t c = 0;
                for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
                    int cnt = 0;
#pragma unroll
                    for (int j = 0; j < kMergeCap / 64; ++j)
                        if (64 * j < n) cnt += __popcll(__ballot(code[j] >= (c | bit)));
                    if (cnt >= a.k) {
                        c |= bit;
                        if (cnt == a.k) break;
                    }
                }
                if (lane == 0) thr = value_of(c);
            }
            __syncthreads();
            t2 = thr;
        }
        // a candidate's place is how many are better: all pairs at once
        if (threadIdx.x == 0) npicked = 0;
        for (int c = threadIdx.x; c < n; c += kMergeThreads) place[c] = 0;
        __syncthreads();
        for (int c = threadIdx.x; c < n; c += kMergeThreads)
            if ((float)list[c].total >= t2) picked[atomicAdd(&npicked, 1)] = c;
        __syncthreads();
        const int m = npicked;
        for (int x = threadIdx.x; x < m * m; x += kMergeThreads) {
            const int me = picked[x / m];
            if (better(list[picked[x % m]], list[me])) atomicAdd(&place[me], 1);
        }
        __syncthreads();
        for (int c = threadIdx.x; c < m; c += kMergeThreads)
            if (place[picked[c]] < a.k) put(place[picked[c]], list[picked[c]]);
        for (int s = n + threadIdx.x; s < a.k; s += kMergeThreads) put_none(s);
        return;
    }
    // more ties than there is room for: the k best one by one, from the lists
    Cand last = {__builtin_huge_val(), 0.f, -1, -1};
    for (int s = 0; s < a.k; ++s) {
        Cand b = {none, 0.f, INT32_MAX, INT32_MAX};
        for (int i = threadIdx.x; i < lists; i += kMergeThreads)
            for (int j = 0; j < a.k; ++j) {
                const int64_t at = (row0 * a.npieces + i) * a.k + j;
                const Cand c = {total_of(i, a.top_v[at]), a.top_v[at], i / a.npieces, a.top_t[at]};
                if (!((float)c.total >= t)) break;
                if (better(last, c)) {
                    if (better(c, b)) b = c;
                    break;  // (the rest of this list is no better)
                }
            }
        if ((int)threadIdx.x < a.nbeam && (float)own[threadIdx.x] >= t) {
            const Cand c = {own[threadIdx.x], 0.f, (int)threadIdx.x, (int)a.eos};
            if (better(last, c) && better(c, b)) b = c;
        }
        __syncthreads();
        list[threadIdx.x] = b;
        __syncthreads();
        for (int d = kMergeThreads / 2; d; d >>= 1) {
            if ((int)threadIdx.x < d && better(list[threadIdx.x + d], list[threadIdx.x]))
                list[threadIdx.x] = list[threadIdx.x + d];
            __syncthreads();
        }
        last = list[0];
        if (threadIdx.x == 0) {
            if (last.beam != INT32_MAX)
                put(s, last);
            else
                put_none(s);
        }
    }
}

struct GatherArgs {
    const int32_t *parents, *tail;
    const char *in;
    char *out;
    int64_t nrows, nin, in_stride, out_stride, bytes;
};

// T: the widest type that every row's start and length allow.  One load that
// waits for another (the parent), then a store: 2 to 5 us with its launch for
// 4 rows of 37 tokens to 512 of 1,023.
template <typename T>
__global__ __launch_bounds__(256) void gather_rows_kernel(GatherArgs a, int64_t chunks) {
    constexpr int64_t kChunk = 256 * 4;  // elements
    const int64_t n = a.bytes / (int64_t)sizeof(T);
    for (int64_t w = blockIdx.x; w < a.nrows * chunks; w += gridDim.x) {
        const int64_t row = w / chunks, x0 = w % chunks * kChunk;
        const int parent = a.parents[row];
        const bool ok = parent >= 0 && parent < a.nin;
        const T *src = (const T *)(a.in + (ok ? parent : 0) * a.in_stride);
        T *dst = (T *)(a.out + row * a.out_stride);
        T v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t x = x0 + i * 256 + threadIdx.x;
            v[i] = T{};
            if (ok && x < n) v[i] = src[x];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t x = x0 + i * 256 + threadIdx.x;
            if (x < n) dst[x] = v[i];
        }
        if (a.tail && x0 == 0 && threadIdx.x == 0)
            *(int32_t *)(a.out + row * a.out_stride + a.bytes) = a.tail[row];
    }
}

template <typename T>
hipError_t launch_gather(const GatherArgs &a, hipStream_t st) {
    const int64_t chunks = std::max<int64_t>(1, (a.bytes / (int64_t)sizeof(T) + 1023) / 1024);
    hipLaunchKernelGGL(gather_rows_kernel<T>, dim3((uint32_t)std::min<int64_t>(a.nrows * chunks, 16384)),
                       dim3(256), 0, st, a, chunks);
    return hipGetLastError();
}

}  // namespace
}  // namespace vs

using vs::report;
using vs::report_hip;

extern "C" {

int vs_beam_create(int device, vs_beam **out) {
    if (!out) return report(VS_ERR_INVALID, "null output handle");
    *out = nullptr;
    int rc = vs::check_device(device);
    if (rc) return rc;
    vs_beam *b = new (std::nothrow) vs_beam();
    if (!b) return report(VS_ERR_OOM, "host allocation");
    b->device = device;
    b->num_cu = vs::cu_count(device);
    *out = b;
    return VS_OK;
}

void vs_beam_destroy(vs_beam *b) {
    if (!b) return;
    vs::DeviceGuard g(b->device);
    (void)hipDeviceSynchronize();
    b->scratch.release();
    delete b;
}

int vs_beam_select(vs_beam *bs, const void *logits, int dtype, int64_t row_stride, int64_t nreq,
                   int64_t nbeam, int64_t vocab, const float *scores, const uint8_t *finished,
                   int64_t eos, int64_t k, float *scores_out, int32_t *tokens_out,
                   int32_t *parents_out, uint8_t *finished_out, void *stream) {
    if (!bs) return report(VS_ERR_INVALID, "null handle");
    if (dtype != VS_DTYPE_F32 && dtype != VS_DTYPE_BF16)
        return report(VS_ERR_INVALID, "unknown dtype code %d", dtype);
    if (nreq < 0 || nbeam <= 0 || vocab <= 0 || k <= 0)
        return report(VS_ERR_INVALID, "nreq must be >= 0, nbeam, vocab and k > 0");
    if (nbeam > vs::kMaxBeams || k > vs::kMaxK)
        return report(VS_ERR_UNSUPPORTED, "nbeam at most %d and k at most %d", vs::kMaxBeams,
                      vs::kMaxK);
    if (vocab > (1 << 30) || nreq > INT32_MAX / nbeam)
        return report(VS_ERR_UNSUPPORTED, "vocab past 2^30 or rows past 2^31");
    if (row_stride < vocab || row_stride > ((int64_t)1 << 40))
        return report(VS_ERR_INVALID, "row_stride %lld below vocab %lld", (long long)row_stride,
                      (long long)vocab);
    if (nreq == 0) return VS_OK;
    if (!logits || !scores || !scores_out || !tokens_out || !parents_out)
        return report(VS_ERR_INVALID, "null buffer");
    const int64_t es = dtype == VS_DTYPE_BF16 ? 2 : 4;
    if ((uintptr_t)logits % es ||
        ((uintptr_t)scores | (uintptr_t)scores_out | (uintptr_t)tokens_out |
         (uintptr_t)parents_out) % 4)
        return report(VS_ERR_INVALID, "a buffer is not aligned to its elements");
    // Requests are merged at once, each from its own scores and flags: another
    // one's outputs must not lie there.
    const struct {
        const void *p;
        int64_t size;
    } ins[] = {{scores, 4}, {finished, 1}},
      outs[] = {{scores_out, 4}, {tokens_out, 4}, {parents_out, 4}, {finished_out, 1}};
    for (const auto &i : ins)
        for (const auto &o : outs) {
            if (i.p == o.p && k == nbeam && i.size == o.size) continue;
            if (vs::overlap(i.p, nreq * nbeam * i.size, o.p, nreq * k * o.size))
                return report(VS_ERR_INVALID, "an output overlaps scores or finished");
        }
    vs::DeviceGuard g(bs->device);
    if (g.err != hipSuccess) return report_hip(g.err, "hipSetDevice");
    hipStream_t st = (hipStream_t)stream;
    vs::BeamArgs a = {};
    a.logits = (const char *)logits;
    a.row_stride = row_stride;
    a.vocab = vocab;
    a.nreq = (int)nreq;
    a.nbeam = (int)nbeam;
    a.k = (int)k;
    // Pieces short enough for 64 waves to a CU, three times what it holds at
    // once: where beams have ended their waves leave at once, and the others
    // spread.  (64 x 8 x 128,000 fp32: 32 waves to a CU 61, 64 58, 128 58 us.)
    // Long steps where 32 waves to a CU have one (bf16, short against long: 16 x
    // 5 x 32,000, k = 10 14.0 and 14.5 us; 30 x 4 x 40,000, k = 4 14.5 and 14.6; 97
    // x 5 x 49,096, k = 10 28.1 and 26.8; 64 x 8 x 128,000, k = 8 43.5 and 40.1).
    const int64_t waves = (int64_t)bs->num_cu * 64;
    const bool is_long = nreq * nbeam * vocab >= (int64_t)bs->num_cu * 32 * 64 * vs::kLongStep;
    const int64_t stretch = 4 * 64 * (is_long ? vs::kLongStep : vs::kShortStep);
    const int64_t row_steps = (vocab + stretch - 1) / stretch * 4;
    a.steps = (int)std::min<int64_t>(vs::kMostSteps,
                                     std::max<int64_t>(1, (nreq * nbeam * row_steps + waves - 1) / waves));
    a.npieces = (int)((row_steps / 4 + a.steps - 1) / a.steps * 4);
    a.scores = scores;
    a.finished = finished;
    a.eos = eos;
    a.scores_out = scores_out;
    a.tokens_out = tokens_out;
    a.parents_out = parents_out;
    a.finished_out = finished_out;
    const int64_t slots = nreq * nbeam * a.npieces;
    if (!vs::grid_ok((slots + 3) / 4, 256) || !vs::grid_ok(nreq, vs::kMergeThreads))
        return report(VS_ERR_UNSUPPORTED, "too many logits or requests");
    void *ws = nullptr;
    int rc = bs->scratch.get(st, (size_t)slots * (sizeof(float2) + (size_t)k * 8), &ws);
    if (rc) return rc;
    a.stat = (float2 *)ws;
    a.top_v = (float *)(a.stat + slots);
    a.top_t = (int32_t *)(a.top_v + slots * k);
    const dim3 grid((uint32_t)((slots + 3) / 4));
    const bool bf16 = dtype == VS_DTYPE_BF16;
    if (is_long && bf16)
        hipLaunchKernelGGL((vs::beam_piece_kernel<1, vs::kLongStep>), grid, dim3(256), 0, st, a);
    else if (is_long)
        hipLaunchKernelGGL((vs::beam_piece_kernel<0, vs::kLongStep>), grid, dim3(256), 0, st, a);
    else if (bf16)
        hipLaunchKernelGGL((vs::beam_piece_kernel<1, vs::kShortStep>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((vs::beam_piece_kernel<0, vs::kShortStep>), grid, dim3(256), 0, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return report_hip(e, "beam select");
    hipLaunchKernelGGL(vs::beam_merge_kernel, dim3((uint32_t)nreq), dim3(vs::kMergeThreads), 0, st, a);
    e = hipGetLastError();
    return e == hipSuccess ? VS_OK : report_hip(e, "beam select");
}

int vs_beam_reorder(vs_beam *bs, const int32_t *parents, int64_t nrows, const void *in,
                    int64_t nrows_in, int64_t in_stride, void *out, int64_t out_stride,
                    int64_t bytes, const int32_t *tail, void *stream) {
    if (!bs) return report(VS_ERR_INVALID, "null handle");
    const int64_t wide = bytes + (tail ? 4 : 0);
    if (nrows < 0 || nrows_in < 0 || bytes < 0 || in_stride < bytes || out_stride < wide)
        return report(VS_ERR_INVALID, "rows of %lld bytes, strides %lld and %lld", (long long)wide,
                      (long long)in_stride, (long long)out_stride);
    if (nrows == 0 || wide == 0) return VS_OK;
    if (!parents || (uintptr_t)parents % 4 || !out || (!in && nrows_in > 0 && bytes > 0))
        return report(VS_ERR_INVALID, "null buffer or unaligned parents");
    if (nrows > INT32_MAX || nrows_in > INT32_MAX)
        return report(VS_ERR_UNSUPPORTED, "more than 2^31 rows");
    if (tail && (((uintptr_t)tail | (uintptr_t)out | (uintptr_t)out_stride | (uintptr_t)bytes) % 4))
        return report(VS_ERR_INVALID, "with tail, out, out_stride and bytes are multiples of 4");
    const int64_t written = (nrows - 1) * out_stride + wide;
    if (vs::overlap(in, nrows_in * in_stride, out, nrows * out_stride))
        return report(VS_ERR_INVALID, "in and out overlap");
    if (vs::overlap(parents, nrows * 4, out, written) || vs::overlap(tail, nrows * 4, out, written))
        return report(VS_ERR_INVALID, "out overlaps parents or tail");
    vs::DeviceGuard g(bs->device);
    if (g.err != hipSuccess) return report_hip(g.err, "hipSetDevice");
    vs::GatherArgs a = {parents,   tail,       (const char *)in, (char *)out, nrows, nrows_in,
                        in_stride, out_stride, bytes};
    hipStream_t st = (hipStream_t)stream;
    const uintptr_t al = (uintptr_t)in | (uintptr_t)out | (uintptr_t)in_stride |
                         (uintptr_t)out_stride | (uintptr_t)bytes;
    hipError_t e;
    if (al % 16 == 0)
        e = vs::launch_gather<u32x4_t>(a, st);
    else if (al % 4 == 0)
        e = vs::launch_gather<uint32_t>(a, st);
    else
        e = vs::launch_gather<uint8_t>(a, st);
    return e == hipSuccess ? VS_OK : report_hip(e, "beam reorder");
}

}  // extern "C"

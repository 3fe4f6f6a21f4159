// vs_logprob.hip -- log probabilities of given tokens, with the entropy of their
// distribution and the likeliest alternatives: kernels and entry point.
#include "vs_logits.h"

namespace vs {
namespace {

constexpr int kMostPieces = 64;  // of a row: one per lane where they are joined
constexpr float kLeast = -1e30f;

struct ScoreArgs {
    const char *logits;
    int64_t row_stride;  // elements
    int64_t vocab;
    int es;              // element size
    int nrows, k, npieces, steps;  // pieces per row, steps per wave and piece
    const int32_t *tokens;
    float *logprob, *entropy;
    int32_t *top_tokens;
    float *top_logprobs;
    float4 *stat;     // [row][piece] maximum m, sums of exp(x - m) and of exp(x - m) (x - m)
    uint64_t *top;    // [row][piece][k] the piece's k largest logits as keys, best first; 0: none
};

// The sums of a distribution about its largest logit, and two of them together.
struct Sums {
    float m, s, w;
};

__device__ __forceinline__ Sums joined(const Sums &a, const Sums &b) {
    const float m = fmaxf(a.m, b.m);
    if (m == VS_NINF) return {m, a.s + b.s, a.w + b.w};
    // (an empty side's maximum is -inf, its sums 0, and 0 times -inf is none)
    const float da = fmaxf(a.m - m, kLeast), db = fmaxf(b.m - m, kLeast);
    const float fa = __builtin_amdgcn_exp2f(da * kLog2e), fb = __builtin_amdgcn_exp2f(db * kLog2e);
    return {m, a.s * fa + b.s * fb, (a.w + a.s * da) * fa + (b.w + b.s * db) * fb};
}

__device__ __forceinline__ Sums shuffled(const Sums &a, int d) {
    return {__shfl_xor(a.m, d), __shfl_xor(a.s, d), __shfl_xor(a.w, d)};
}

// What a row's sums say.  log sum exp is m + log s; the entropy is log s - w / s;
// in this order no size of the logits costs them digits.  A row that holds a NaN
// or +inf, or nothing but -inf, has no distribution: s is a NaN or 0.
struct Row {
    double off;  // log s; NaN: no distribution
    float m;
};

__device__ __forceinline__ Row finish_row(const ScoreArgs &a, int row, const Sums &t, bool first) {
    Row r;
    r.m = t.m;
    r.off = t.s > 0.f ? log((double)t.s) : __builtin_nan("");
    if (first) {
        if (a.entropy) a.entropy[row] = (float)(r.off - (double)t.w / (double)t.s);
        if (a.logprob) {
            const int token = a.tokens[row];
            double lp = __builtin_nan("");
            if (token >= 0 && token < a.vocab) lp = 0.0;
            if (lp == 0.0) {
                const int64_t at = row * a.row_stride + token;
                const float x = a.es == 2 ? float_of((uint32_t)((const uint16_t *)a.logits)[at] << 16)
                                          : ((const float *)a.logits)[at];
                lp = ((double)x - (double)t.m) - r.off;
            }
            a.logprob[row] = token == -1 ? 0.f : (float)lp;
        }
    }
    return r;
}

// One pass over the logits: a workgroup takes a piece of a row, its waves the steps
// of 64 PER logits in turn.  Per logit one exponential and two sums.  The list of
// the k largest is beam search's: what is at or above a threshold that k logits
// seen so far reach.  Bound by HBM: 2,048 x 128,000 in bf16 92 us (5.7 TB/s of the 6.3
// that a plain read reaches), 1,024 x 64,000 in fp32 44 us with its join (6.0); 20 x
// 50,001 with k = 5 by latency, 7 us.  Lists add their thresholds' instructions: k = 5 and
// 20 114 and 132 us, 51 and 67 (k = 0 97 and 44, joins included).  fp32's long steps are held to four waves a SIMD:
// with six they spill 90 registers.
template <int ST, int PER, bool TOP>
__global__ __launch_bounds__(256, PER == kLongStep ? (ST ? 6 : 4) : 1) void logprob_piece_kernel(ScoreArgs a) {
    using S = Step<ST, PER>;
    constexpr int kStep = 64 * PER, kNext = 4 * kStep;
    __shared__ uint64_t lists[TOP ? 4 : 1][TOP ? kCap : 1];
    __shared__ Sums sums[4];
    __shared__ int counts[4];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint64_t *cand = lists[TOP ? wave : 0];
    const int row = blockIdx.x / (uint32_t)a.npieces, piece = blockIdx.x % (uint32_t)a.npieces;
    const char *base = a.logits + row * a.row_stride * S::ES;
    const int vocab = (int)a.vocab;
    const int64_t stretch = (int64_t)a.steps * kNext;
    const int64_t begin = piece * stretch + wave * kStep;
    const int64_t end = min((piece + 1) * stretch, (int64_t)vocab);

    float run = VS_NINF;  // the lane's maximum so far
    float top = VS_NINF;  // the wave's
    float sum = 0.f, weighted = 0.f;  // of exp(x - top) and exp(x - top) (x - top), the lane's share
    float thr = -__FLT_MAX__;         // (so -inf is no candidate)
    int n = 0;
    S step;
    if (begin < end) step.load(base, (int)begin, vocab, lane);
    for (int64_t first = begin; first < end; first += kNext) {
        const S x = step;
        if (PER == kShortStep && first + kNext < end) step.load(base, (int)(first + kNext), vocab, lane);
        float most = fmaxf(x.value(0), x.value(1));
#pragma unroll
        for (int i = 2; i < PER; i += 2) most = max3(most, x.value(i), x.value(i + 1));
        if (__ballot(most > top)) {
            const float m = wave_max(most);
            const float d = fmaxf(top - m, kLeast), f = __builtin_amdgcn_exp2f(d * kLog2e);
            weighted = (weighted + sum * d) * f;
            sum *= f;
            top = m;
        }
        if (TOP && __ballot(most >= thr)) {
            run = fmaxf(run, most);
            // the k-th largest of the lanes' maxima: no lower than the last one,
            // whose leading bits that the largest has too are its
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
            if (t > low) thr = value_of(t);
            const int n0 = n;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const float v = x.value(i);
                const uint64_t in = __ballot(v >= thr);
                if (in) {
                    const int at = n + below(in);
                    if (v >= thr && at < kCap) cand[at] = key_of(v, S::token((int)first, i, lane));
                    n += __popcll(in);
                }
            }
            if (n > kCap) {
                // more than the list holds, ties mostly: again, a register at a
                // time, cut to the k best in between.  What ties with the k-th of
                // these in a later step has a higher token and is out.
                n = n0;
#pragma unroll 1
                for (int i = 0; i < PER; ++i) {
                    const float v = S::reload(base, (int)first, i, vocab, lane);
                    const uint64_t in = __ballot(v >= thr);
                    if (!in) continue;
                    if (n > kCap - 64) {
                        cut_list(cand, n, a.k, lane);
                        n = min(n, a.k);
                    }
                    if (v >= thr) cand[n + below(in)] = key_of(v, S::token((int)first, i, lane));
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
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const float d = x.value(i) - ref, e = __builtin_amdgcn_exp2f(d * kLog2e);
            sum += e;
            t = __builtin_fmaf(e, d, t);
        }
        if (__ballot(t != t)) {  // -inf among them, times a weight of 0 (or a NaN, which stays one)
            t = 0.f;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const float d = x.value(i) - ref, e = __builtin_amdgcn_exp2f(d * kLog2e);
                t = __builtin_fmaf(e, fmaxf(d, kLeast), t);
            }
        }
        weighted += t;
        if (PER != kShortStep && first + kNext < end) step.load(base, (int)(first + kNext), vocab, lane);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        sum += __shfl_xor(sum, d);
        weighted += __shfl_xor(weighted, d);
    }
    if (lane == 0) sums[wave] = {top, sum, weighted};
    if (TOP) {
        cut_list(cand, n, a.k, lane);
        if (lane == 0) counts[wave] = min(n, a.k);
    }
    __syncthreads();
    const Sums all = joined(joined(sums[0], sums[1]), joined(sums[2], sums[3]));
    const int64_t slot = blockIdx.x;
    Row r = {0.0, 0.f};
    if (a.npieces == 1)
        r = finish_row(a, row, all, threadIdx.x == 0);
    else if (threadIdx.x == 0)
        a.stat[slot] = make_float4(all.m, all.s, all.w, 0.f);
    if constexpr (TOP) {
        // the waves' lists in one: an entry's place is how many are better
        int have = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) have += counts[w];
        auto put = [&](int at, uint64_t key) {
            if (a.npieces > 1) {
                a.top[slot * a.k + at] = key;
            } else {
                const bool some = key && r.off == r.off;
                a.top_tokens[(int64_t)row * a.k + at] = some ? (int)~(uint32_t)key : -1;
                a.top_logprobs[(int64_t)row * a.k + at] =
                    some ? (float)(((double)value_of((uint32_t)(key >> 32)) - (double)r.m) - r.off)
                         : VS_NINF;
            }
        };
        if ((int)threadIdx.x < 4 * a.k) {
            const int w = threadIdx.x / a.k, i = threadIdx.x % a.k;
            if (i < counts[w]) {
                const uint64_t me = lists[w][i];
                int rank = i;  // (a list is in order)
                for (int v = 0; v < 4; ++v)
                    if (v != w)
                        for (int j = 0; j < counts[v]; ++j) rank += lists[v][j] > me;
                if (rank < a.k) put(rank, me);
            }
        }
        for (int at = have + threadIdx.x; at < a.k; at += 256) put(at, 0);
    }
}

// A wave per row joins its pieces: their sums, and their lists, of which the best
// first entry is taken k times.  4 to 5 us, latency.
__global__ __launch_bounds__(256) void logprob_join_kernel(ScoreArgs a) {
    const int lane = threadIdx.x & 63;
    const int row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (row >= a.nrows) return;
    Sums t = {VS_NINF, 0.f, 0.f};
    const bool mine = lane < a.npieces;
    const uint64_t *list = a.top + ((int64_t)row * a.npieces + lane) * a.k;
    uint64_t head = 0;
    if (mine) {
        const float4 x = a.stat[(int64_t)row * a.npieces + lane];
        t = {x.x, x.y, x.z};
        if (a.k) head = list[0];
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) t = joined(t, shuffled(t, d));
    const Row r = finish_row(a, row, t, lane == 0);
    if (!a.k) return;
    int at = 0;
    int32_t token = -1;  // lane i keeps the i-th of the k best
    float value = 0.f;
    for (int i = 0; i < a.k; ++i) {
        const uint32_t high = (uint32_t)(head >> 32);
        // (codes are compared as the floats that they stand for; none is a NaN)
        const float best = wave_max(high ? value_of(high) : VS_NINF);
        uint64_t in = __ballot(high != 0 && value_of(high) == best);
        if (!in) break;
        int l = __builtin_ctzll(in);
        uint32_t low = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)head, l);
        for (in &= in - 1; in; in &= in - 1) {  // equal logits: the lowest token
            const int o = __builtin_ctzll(in);
            const uint32_t other = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)head, o);
            if (other > low) {
                low = other;
                l = o;
            }
        }
        if (lane == i) {
            token = (int)~low;
            value = best;
        }
        if (lane == l) head = ++at < a.k ? list[at] : 0;
    }
    if (lane < a.k) {
        const bool some = token >= 0 && r.off == r.off;
        a.top_tokens[(int64_t)row * a.k + lane] = some ? token : -1;
        a.top_logprobs[(int64_t)row * a.k + lane] =
            some ? (float)(((double)value - (double)r.m) - r.off) : VS_NINF;
    }
}

template <int ST, int PER>
void launch_pieces(const ScoreArgs &a, hipStream_t st) {
    const dim3 grid((uint32_t)a.nrows * (uint32_t)a.npieces);
    if (a.k)
        hipLaunchKernelGGL((logprob_piece_kernel<ST, PER, true>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((logprob_piece_kernel<ST, PER, false>), grid, dim3(256), 0, st, a);
}

}  // namespace
}  // namespace vs

using vs::report;
using vs::report_hip;

extern "C" {

int vs_beam_logprobs(vs_beam *bs, const void *logits, int dtype, int64_t row_stride, int64_t nrows,
                     int64_t vocab, const int32_t *tokens, float *logprobs, float *entropy,
                     int64_t k, int32_t *top_tokens, float *top_logprobs, void *stream) {
    if (!bs) return report(VS_ERR_INVALID, "null handle");
    if (dtype != VS_DTYPE_F32 && dtype != VS_DTYPE_BF16)
        return report(VS_ERR_INVALID, "unknown dtype code %d", dtype);
    if (nrows < 0 || vocab <= 0 || k < 0)
        return report(VS_ERR_INVALID, "nrows and k must be >= 0, vocab > 0");
    if (k > vs::kMaxK) return report(VS_ERR_UNSUPPORTED, "k at most %d", vs::kMaxK);
    if (vocab > (1 << 30) || nrows > INT32_MAX)
        return report(VS_ERR_UNSUPPORTED, "vocab past 2^30 or rows past 2^31");
    if (row_stride < vocab || row_stride > ((int64_t)1 << 40))
        return report(VS_ERR_INVALID, "row_stride %lld below vocab %lld", (long long)row_stride,
                      (long long)vocab);
    if (!tokens != !logprobs)
        return report(VS_ERR_INVALID, "tokens and logprobs are given together or not at all");
    if (nrows == 0) return VS_OK;
    if (!logits || (k && (!top_tokens || !top_logprobs)))
        return report(VS_ERR_INVALID, "null buffer");
    const int64_t es = dtype == VS_DTYPE_BF16 ? 2 : 4;
    if ((uintptr_t)logits % es || ((uintptr_t)tokens | (uintptr_t)logprobs | (uintptr_t)entropy |
                                   (uintptr_t)(k ? top_tokens : nullptr) |
                                   (uintptr_t)(k ? top_logprobs : nullptr)) % 4)
        return report(VS_ERR_INVALID, "a buffer is not aligned to its elements");
    // Rows are finished while others are read.
    const struct {
        const void *p;
        int64_t size;
    } outs[] = {{logprobs, nrows * 4}, {entropy, nrows * 4}, {k ? top_tokens : nullptr, nrows * k * 4},
                {k ? top_logprobs : nullptr, nrows * k * 4}};
    for (int i = 0; i < 4; ++i) {
        if (vs::overlap(logits, ((nrows - 1) * row_stride + vocab) * es, outs[i].p, outs[i].size) ||
            vs::overlap(tokens, nrows * 4, outs[i].p, outs[i].size))
            return report(VS_ERR_INVALID, "an output overlaps logits or tokens");
        for (int j = 0; j < i; ++j)
            if (vs::overlap(outs[i].p, outs[i].size, outs[j].p, outs[j].size))
                return report(VS_ERR_INVALID, "two outputs overlap");
    }
    vs::DeviceGuard g(bs->device);
    if (g.err != hipSuccess) return report_hip(g.err, "hipSetDevice");
    hipStream_t st = (hipStream_t)stream;
    vs::ScoreArgs a = {};
    a.logits = (const char *)logits;
    a.es = (int)es;
    a.row_stride = row_stride;
    a.vocab = vocab;
    a.nrows = (int)nrows;
    a.k = (int)k;
    a.tokens = tokens;
    a.logprob = logprobs;
    a.entropy = entropy;
    a.top_tokens = top_tokens;
    a.top_logprobs = top_logprobs;
    // Rows are divided where there are fewer than 16 workgroups to a CU.
    const bool is_long = nrows * vocab >= (int64_t)bs->num_cu * 32 * 64 * vs::kLongStep;
    const int64_t stretch = 4 * 64 * (is_long ? vs::kLongStep : vs::kShortStep);
    const int64_t row_steps = (vocab + stretch - 1) / stretch;
    int64_t pieces = std::min<int64_t>({row_steps, vs::kMostPieces,
                                        std::max<int64_t>(1, (int64_t)bs->num_cu * 16 / nrows)});
    const int64_t steps = (row_steps + pieces - 1) / pieces;
    pieces = (row_steps + steps - 1) / steps;
    a.steps = (int)steps;
    a.npieces = (int)pieces;
    if (!vs::grid_ok(nrows * pieces, 256))
        return report(VS_ERR_UNSUPPORTED, "%lld rows", (long long)nrows);
    if (pieces > 1) {
        void *ws = nullptr;
        int rc = bs->scratch.get(st, (size_t)(nrows * pieces) * (sizeof(float4) + (size_t)k * 8), &ws);
        if (rc) return rc;
        a.stat = (float4 *)ws;
        a.top = (uint64_t *)(a.stat + nrows * pieces);
    }
    if (is_long && es == 2)
        vs::launch_pieces<1, vs::kLongStep>(a, st);
    else if (is_long)
        vs::launch_pieces<0, vs::kLongStep>(a, st);
    else if (es == 2)
        vs::launch_pieces<1, vs::kShortStep>(a, st);
    else
        vs::launch_pieces<0, vs::kShortStep>(a, st);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && pieces > 1) {
        hipLaunchKernelGGL(vs::logprob_join_kernel, dim3((uint32_t)((nrows + 3) / 4)), dim3(256), 0, st, a);
        e = hipGetLastError();
    }
    return e == hipSuccess ? VS_OK : report_hip(e, "log probabilities");
}

}  // extern "C"

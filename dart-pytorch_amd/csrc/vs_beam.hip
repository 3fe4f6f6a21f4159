// vs_beam.hip -- beam search: the choice of the next beams over beams and
// vocabulary, and the reordering of their states.
#include "vs_host.h"
#include "vs_internal.h"

struct vs_beam {
    int device = 0;
    vs::StreamScratch scratch;
};

namespace vs {
namespace {

constexpr int kMaxK = 64, kMaxBeams = 128;
constexpr int kPiece = 2048;   // logits per wave: 32 per lane, held in registers
constexpr int kCap = 256;      // candidates per piece kept in LDS
constexpr int kMergeCap = 1024;
constexpr float kLog2e = 1.44269504088896340736f;
#define VS_NINF (-__builtin_huge_valf())

struct BeamArgs {
    const char *logits;
    int64_t row_stride;  // elements
    int64_t vocab;
    int nreq, nbeam, k, npieces;
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

// larger float, larger code; neither infinity nor -0 needs a case of its own
__device__ __forceinline__ uint32_t code_of(float x) {
    const uint32_t u = bits_of(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t c) {
    return float_of(c & 0x80000000u ? c & 0x7FFFFFFFu : ~c);
}

// One pass over the logits: a wave loads its piece of a row once and leaves
// the piece's maximum and exponential sum (for the row's log sum exp) and its
// k largest logits.  A threshold that k logits are at or above is the k-th
// largest of the lanes' maxima, found by bisection on ballots; what lies at or
// above it, a few more than k, is ranked through LDS.  Only where more than
// kCap logits tie at the threshold are the k best picked one by one.
template <int ST>
__global__ __launch_bounds__(256) void beam_piece_kernel(BeamArgs a) {
    constexpr int E = ST ? 8 : 4, NL = 32 / E, ES = 16 / E;
    __shared__ float cand_v[4][kCap];
    __shared__ int cand_t[4][kCap];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t slot = (int64_t)blockIdx.x * 4 + wave;
    if (slot >= (int64_t)a.nreq * a.nbeam * a.npieces) return;
    const int64_t row = slot / a.npieces;
    const int piece = (int)(slot % a.npieces);
    // a beam without continuations of its own: its logits do not matter
    const float score = a.scores[row];
    if (!(score > VS_NINF) || (a.finished && a.finished[row])) return;
    const char *base = a.logits + row * a.row_stride * ES;
    const int first = piece * kPiece;

    // (which lane holds which token goes by the token alone, wherever the row
    // starts: equal rows have equal sums to the bit, and their beams tie)

    float x[32];
    if (first + kPiece <= a.vocab) {
#pragma unroll
        for (int l = 0; l < NL; ++l) {
            u32x4_t w;
            __builtin_memcpy(&w, base + (int64_t)(first + (l * 64 + lane) * E) * ES, 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (ST) {
                    x[l * E + 2 * i] = float_of(w[i] << 16);
                    x[l * E + 2 * i + 1] = float_of(w[i] & 0xFFFF0000u);
                } else {
                    x[l * E + i] = float_of(w[i]);
                }
            }
        }
    } else {
        // the row's last, partial piece: one load per token, all in flight
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const int64_t t = first + ((i / E) * 64 + lane) * E + i % E;
            const int64_t at = min(t, a.vocab - 1);
            float v;
            if constexpr (ST)
                v = bf16_to_f32(((const uint16_t *)base)[at]);
            else
                v = ((const float *)base)[at];
            x[i] = t < a.vocab ? v : VS_NINF;
        }
    }
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 32; ++i) top = fmaxf(top, x[i]);
    top = top > VS_NINF ? top : VS_NINF;  // (all NaN)
    float wtop = top;
#pragma unroll
    for (int d = 32; d; d >>= 1) wtop = fmaxf(wtop, __shfl_xor(wtop, d));
    const float ref = wtop == VS_NINF ? 0.f : wtop;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) sum += __builtin_amdgcn_exp2f((x[i] - ref) * kLog2e);
#pragma unroll
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    if (lane == 0) a.stat[slot] = make_float2(wtop, sum);

    const uint32_t code = code_of(top);
    uint32_t thr = 0;
    for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
        const int cnt = __popcll(__ballot(code >= (thr | bit)));
        if (cnt >= a.k) {
            thr |= bit;
            if (cnt == a.k) break;
        }
    }
    const float tv = value_of(thr);
    // (the bisection ends below -inf's code only if that lane's maximum is
    // smaller still, which none is)
    int n = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const bool in = x[i] > VS_NINF && !(x[i] < tv);
        const uint64_t mask = __ballot(in);
        if (mask) {
            const int at = n + __popcll(mask & (((uint64_t)1 << lane) - 1));
            if (in && at < kCap) {
                cand_v[wave][at] = x[i];
                cand_t[wave][at] = first + ((i / E) * 64 + lane) * E + i % E;
            }
            n += __popcll(mask);
        }
    }
    float *ov = a.top_v + slot * a.k;
    int32_t *ot = a.top_t + slot * a.k;
    if (n <= kCap) {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
        for (int c = lane; c < n; c += 64) {
            const float v = cand_v[wave][c];
            const int t = cand_t[wave][c];
            int rank = 0;
            for (int j = 0; j < n; ++j) {
                const float vj = cand_v[wave][j];
                rank += vj > v || (vj == v && cand_t[wave][j] < t);
            }
            if (rank < a.k) {
                ov[rank] = v;
                ot[rank] = t;
            }
        }
        for (int c = n + lane; c < a.k; c += 64) {
            ov[c] = VS_NINF;
            ot[c] = -1;
        }
        return;
    }
    float lv = __builtin_huge_valf();
    int lt = -1;  // the last one picked
    for (int s = 0; s < a.k; ++s) {
        float bv = VS_NINF;
        int bt = INT32_MAX;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const int t = first + ((i / E) * 64 + lane) * E + i % E;
            const bool after = x[i] < lv || (x[i] == lv && t > lt);
            if (after && x[i] > VS_NINF && (x[i] > bv || (x[i] == bv && t < bt))) {
                bv = x[i];
                bt = t;
            }
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) {
            const float v = __shfl_xor(bv, d);
            const int t = __shfl_xor(bt, d);
            if (v > bv || (v == bv && t < bt)) {
                bv = v;
                bt = t;
            }
        }
        if (lane == 0) {
            ov[s] = bv;
            ot[s] = bt == INT32_MAX ? -1 : bt;
        }
        lv = bv;
        lt = bt;
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
// k best of the pieces' candidates, in 64 bits.  The pieces' lists are sorted,
// so the threshold (the k-th largest of the threads' best heads) needs their
// first entries only and each list is walked no further than it.
__global__ __launch_bounds__(256) void beam_merge_kernel(BeamArgs a) {
    // total = (logit - largest) + (score - log of the sum of exponentials): in
    // this order no size of the logits costs the total its digits
    __shared__ double offset[kMaxBeams];  // score - log sum; NaN: no candidates
    __shared__ float largest[kMaxBeams];
    __shared__ double best[256];
    __shared__ Cand list[kMergeCap];
    __shared__ int nlist;
    __shared__ double thr;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = blockIdx.x;
    const int64_t row0 = (int64_t)r * a.nbeam;
    const double none = -__builtin_huge_val();
    for (int w = wave; w < a.nbeam; w += 4) {
        const int64_t row = row0 + w;
        const float score = a.scores[row];
        const bool live = score > VS_NINF && !(a.finished && a.finished[row]);
        double off = __builtin_nan("");
        if (live) {
            const float2 *st = a.stat + row * a.npieces;
            float top = VS_NINF;
            for (int p = lane; p < a.npieces; p += 64) top = fmaxf(top, st[p].x);
#pragma unroll
            for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
            const float ref = top == VS_NINF ? 0.f : top;
            double sum = 0.0;
            for (int p = lane; p < a.npieces; p += 64)
                sum += (double)st[p].y * (double)__builtin_amdgcn_exp2f((st[p].x - ref) * kLog2e);
#pragma unroll
            for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
            // (a NaN or +inf among the logits makes the sum a NaN; nothing but -inf makes it 0)
            if (sum > 0.0) off = (double)score - log(sum);
            if (lane == 0) largest[w] = top;
        }
        if (lane == 0) offset[w] = off;
    }
    if (threadIdx.x == 0) nlist = 0;
    __syncthreads();

    // candidate `c` of list (w, p), or nothing
    auto fetch = [&](int w, int p, int c, Cand &out) {
        const double off = offset[w];
        if (off != off) return false;
        const int64_t at = ((row0 + w) * a.npieces + p) * a.k + c;
        out.v = a.top_v[at];
        if (!(out.v > VS_NINF)) return false;
        out.token = a.top_t[at];
        out.beam = w;
        out.total = off + ((double)out.v - (double)largest[w]);
        return true;
    };
    auto ended = [&](int w, Cand &out) {
        const int64_t row = row0 + w;
        const float score = a.scores[row];
        if (!(score > VS_NINF) || !a.finished || !a.finished[row]) return false;
        if (a.eos < 0 || a.eos >= a.vocab) return false;
        out.total = (double)score;
        out.v = 0.f;
        out.beam = w;
        out.token = (int)a.eos;
        return true;
    };
    const int lists = a.nbeam * a.npieces;
    double mine = none;
    for (int i = threadIdx.x; i < lists; i += 256) {
        Cand c;
        if (fetch(i / a.npieces, i % a.npieces, 0, c)) mine = max(mine, c.total);
    }
    for (int w = threadIdx.x; w < a.nbeam; w += 256) {
        Cand c;
        if (ended(w, c)) mine = max(mine, c.total);
    }
    best[threadIdx.x] = mine;
    __syncthreads();
    int rank = 0;
    for (int i = 0; i < 256; ++i) {
        const double o = best[i];
        rank += o > mine || (o == mine && i < (int)threadIdx.x);
    }
    if (rank == a.k - 1) thr = mine;
    __syncthreads();
    const double t = thr;
    for (int i = threadIdx.x; i < lists; i += 256)
        for (int j = 0; j < a.k; ++j) {
            Cand c;
            if (!fetch(i / a.npieces, i % a.npieces, j, c) || c.total < t) break;
            const int at = atomicAdd(&nlist, 1);
            if (at >= kMergeCap) break;
            list[at] = c;
        }
    for (int w = threadIdx.x; w < a.nbeam; w += 256) {
        Cand c;
        if (ended(w, c) && !(c.total < t)) {
            const int at = atomicAdd(&nlist, 1);
            if (at < kMergeCap) list[at] = c;
        }
    }
    __syncthreads();
    const int n = nlist;
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
    if (n <= kMergeCap) {
        for (int c = threadIdx.x; c < n; c += 256) {
            const Cand me = list[c];
            int rk = 0;
            for (int j = 0; j < n; ++j) rk += better(list[j], me);
            if (rk < a.k) put(rk, me);
        }
        for (int s = n + threadIdx.x; s < a.k; s += 256) put_none(s);
        return;
    }
    // more ties than the list holds: one by one
    Cand last;
    last.total = __builtin_huge_val();
    last.beam = -1;
    last.v = 0.f;
    last.token = -1;
    for (int s = 0; s < a.k; ++s) {
        Cand b;
        b.total = none;
        b.beam = INT32_MAX;
        b.v = 0.f;
        b.token = INT32_MAX;
        for (int i = threadIdx.x; i < lists; i += 256)
            for (int j = 0; j < a.k; ++j) {
                Cand c;
                if (!fetch(i / a.npieces, i % a.npieces, j, c) || c.total < t) break;
                if (better(last, c)) {
                    if (better(c, b)) b = c;
                    break;  // (the rest of this list is no better)
                }
            }
        for (int w = threadIdx.x; w < a.nbeam; w += 256) {
            Cand c;
            if (ended(w, c) && better(last, c) && better(c, b)) b = c;
        }
        __syncthreads();
        list[threadIdx.x] = b;
        __syncthreads();
        for (int d = 128; d; d >>= 1) {
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

// T: the widest type that every row's start and length allow.
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
    a.npieces = (int)((vocab + vs::kPiece - 1) / vs::kPiece);
    a.scores = scores;
    a.finished = finished;
    a.eos = eos;
    a.scores_out = scores_out;
    a.tokens_out = tokens_out;
    a.parents_out = parents_out;
    a.finished_out = finished_out;
    const int64_t slots = nreq * nbeam * a.npieces;
    if ((slots + 3) / 4 > INT32_MAX) return report(VS_ERR_UNSUPPORTED, "too many logits");
    void *ws = nullptr;
    int rc = bs->scratch.get(st, (size_t)slots * (sizeof(float2) + (size_t)k * 8), &ws);
    if (rc) return rc;
    a.stat = (float2 *)ws;
    a.top_v = (float *)(a.stat + slots);
    a.top_t = (int32_t *)(a.top_v + slots * k);
    const dim3 grid((uint32_t)((slots + 3) / 4));
    if (dtype == VS_DTYPE_BF16)
        hipLaunchKernelGGL(vs::beam_piece_kernel<1>, grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL(vs::beam_piece_kernel<0>, grid, dim3(256), 0, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return report_hip(e, "beam select");
    hipLaunchKernelGGL(vs::beam_merge_kernel, dim3((uint32_t)nreq), dim3(256), 0, st, a);
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
    const char *i0 = (const char *)in, *o0 = (const char *)out;
    if (in && i0 < o0 + nrows * out_stride && o0 < i0 + nrows_in * in_stride)
        return report(VS_ERR_INVALID, "in and out overlap");
    vs::DeviceGuard g(bs->device);
    if (g.err != hipSuccess) return report_hip(g.err, "hipSetDevice");
    vs::GatherArgs a = {parents,   tail,       i0, (char *)out, nrows, nrows_in,
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

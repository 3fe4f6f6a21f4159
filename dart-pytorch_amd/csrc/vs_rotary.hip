// vs_rotary.hip -- rotary positions: rows of queries and keys turned by angles
// that grow with their positions, by themselves and on the way into the paged
// cache: kernels and entry points.
#include <cmath>

#include "vs_rows.h"

struct vs_rotary {
    int device = 0;
    int dims = 0;
    bool interleaved = false;
    float gain = 1.f;
    uint64_t *turns = nullptr;  // [dims / 2] turns per position, in units of 2^-64
    int num_cu = 256;
};

namespace vs {
namespace {

// The turn of one pair: y0 = x0 cos - x1 sin, y1 = x1 cos + x0 sin, cosine and
// sine times the gain.
struct Turn {
    float c, s;
};

// Angles are whole numbers of 2^-64 turns, so their product with a position wraps
// at whole turns by itself and is exact however far the position is; what is
// rounded is the frequency, once, to 2^-64 turns per position.  Of the product the
// nearest quarter turn is taken off; the rest, at most an eighth of a turn, becomes
// an fp32 angle with both of its words (the upper one alone would cut off up to
// 2^-32 of a turn, all of a small angle) and goes through the Taylor polynomials of
// sine and cosine, whose first terms left out are (pi/4)^11 / 11! = 1.8e-9 and
// (pi/4)^12 / 12! = 1.2e-10.
__device__ __forceinline__ Turn turn_of(uint64_t phase, float gain) {
    const uint32_t u = (uint32_t)(phase >> 32);
    const uint32_t quarter = (u + 0x20000000u) >> 30;
    const float x = __builtin_fmaf((float)(uint32_t)phase, (float)(6.283185307179586 * 0x1p-64),
                                   (float)(int32_t)(u - (quarter << 30)) * (float)(6.283185307179586 * 0x1p-32));
    const float x2 = x * x;
    float s = 1.f / 362880.f, c = -1.f / 3628800.f;
    s = __builtin_fmaf(s, x2, -1.f / 5040.f);
    s = __builtin_fmaf(s, x2, 1.f / 120.f);
    s = __builtin_fmaf(s, x2, -1.f / 6.f);
    s = __builtin_fmaf(s * x2, x, x);
    c = __builtin_fmaf(c, x2, 1.f / 40320.f);
    c = __builtin_fmaf(c, x2, -1.f / 720.f);
    c = __builtin_fmaf(c, x2, 1.f / 24.f);
    c = __builtin_fmaf(c, x2, -0.5f);
    c = __builtin_fmaf(c, x2, 1.f);
    // a quarter turn on: (c, s) -> (-s, c)
    const bool odd = quarter & 1;
    const float a = odd ? s : c, b = odd ? c : s;
    const uint32_t sc = (quarter + 1) << 30 & 0x80000000u, ss = quarter << 30 & 0x80000000u;
    return {float_of(bits_of(a) ^ sc) * gain, float_of(bits_of(b) ^ ss) * gain};
}

// (the rounding of the second product is the only one besides the result's)
__device__ __forceinline__ void turn_pair(const Turn &t, float &x0, float &x1) {
    const float y0 = __builtin_fmaf(x0, t.c, -(x1 * t.s));
    x1 = __builtin_fmaf(x1, t.c, x0 * t.s);
    x0 = y0;
}

template <int ST>
__device__ __forceinline__ float value_at(const u32x4_t &w, int i) {
    if constexpr (ST) {
        const uint32_t x = w[i / 2];
        return float_of(i % 2 ? x & 0xFFFF0000u : x << 16);
    } else {
        return float_of(w[i]);
    }
}

template <int ST>
__device__ __forceinline__ u32x4_t pack(const float *x) {
    u32x4_t w;
    if constexpr (ST) {
        bf16x8_t y;
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = (__bf16)x[i];
        w = __builtin_bit_cast(u32x4_t, y);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = bits_of(x[i]);
    }
    return w;
}

struct RotaryArgs {
    const uint64_t *turns;
    float gain;
    int dims, interleaved;
};

// A row's rotated part comes in units of E pairs (VEC: two 16-byte pieces), or of
// one pair where rows or the part do not divide into such pieces.
template <int ST, bool VEC>
struct Unit {
    static constexpr int E = ST ? 8 : 4;
    static constexpr int N = VEC ? E : 1;
    using T = typename std::conditional<ST, uint16_t, uint32_t>::type;
    Turn t[N];
    int at0, at1;  // its first elements: of two pieces, or of a pair

    __device__ __forceinline__ void angles(const RotaryArgs &r, int u, int64_t pos) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            t[i] = turn_of((uint64_t)pos * r.turns[u * N + i], r.gain);
        at0 = r.interleaved ? 2 * N * u : N * u;
        at1 = at0 + (r.interleaved ? N : r.dims / 2);
    }
    // The unit of `row`, turned: the pieces' new contents.
    __device__ __forceinline__ void apply(const RotaryArgs &r, const T *row, u32x4_t &w0,
                                          u32x4_t &w1) const {
        if constexpr (VEC) {
            w0 = *(const u32x4_t *)(row + at0);
            w1 = *(const u32x4_t *)(row + at1);
            float x[2 * N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                x[i] = value_at<ST>(w0, i);
                x[N + i] = value_at<ST>(w1, i);
            }
            if (r.interleaved) {
#pragma unroll
                for (int i = 0; i < N; ++i) turn_pair(t[i], x[2 * i], x[2 * i + 1]);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) turn_pair(t[i], x[i], x[N + i]);
            }
            w0 = pack<ST>(x);
            w1 = pack<ST>(x + N);
        } else {
            float x0, x1;
            if constexpr (ST) {
                x0 = float_of((uint32_t)row[at0] << 16);
                x1 = float_of((uint32_t)row[at1] << 16);
            } else {
                x0 = float_of(row[at0]);
                x1 = float_of(row[at1]);
            }
            turn_pair(t[0], x0, x1);
            if constexpr (ST) {
                w0[0] = __builtin_bit_cast(uint16_t, (__bf16)x0);
                w1[0] = __builtin_bit_cast(uint16_t, (__bf16)x1);
            } else {
                w0[0] = bits_of(x0);
                w1[0] = bits_of(x1);
            }
        }
    }
    static __device__ __forceinline__ void store(T *to, const u32x4_t &w) {
        if constexpr (VEC)
            *(u32x4_t *)to = w;
        else
            *to = (T)w[0];
    }
};

struct TurnArgs {
    RotaryArgs r;
    const char *x;
    char *out;
    const int32_t *positions;
    int64_t x_row, x_head, o_row, o_head, nrows;
    int heads, dim;
    int copy, back;  // the rest of the head goes to another place; the other way round
};

// Rows by themselves.  A thread turns one unit of a row in every `spread`-th head,
// so that its angles are computed once for several heads and neighbouring
// threads read neighbouring bytes.  Bound by HBM: 8,192 rows of 32 heads of 128 in bf16
// 25.4 us (134 MB read and written, 5.3 TB/s) either way round, interleaved and in place
// too, in fp32 43 (6.2); a quarter of the head turned in place 8.0 and 9.2.  Single pairs,
// where rows or parts do not divide into pieces: 8,191 rows of 13 heads of 80, 20 of them
// turned, 21 us.  64 rows 6.5, launch and latency.
template <int ST, bool VEC>
__global__ __launch_bounds__(256) void rotate_kernel(TurnArgs a, int spread) {
    using U = Unit<ST, VEC>;
    using T = typename U::T;
    constexpr int P = VEC ? U::E : 1;  // elements of a piece
    const int units = a.r.dims / 2 / U::N, rest = a.copy ? (a.dim - a.r.dims) / P : 0;
    const int64_t each = (int64_t)spread * (units + rest);
    const int64_t stride = (int64_t)gridDim.x * 256;
    for (int64_t w = (int64_t)blockIdx.x * 256 + threadIdx.x; w < a.nrows * each; w += stride) {
        const int64_t row = w / each;
        const int in = (int)(w % each), u = in % (units + rest);
        const T *x = (const T *)a.x + row * a.x_row;
        T *out = (T *)a.out + row * a.o_row;
        if (u < units) {
            U t;
            const int64_t pos = a.positions[row];
            t.angles(a.r, u, a.back ? -pos : pos);
            for (int h = in / (units + rest); h < a.heads; h += spread) {
                u32x4_t w0, w1;
                t.apply(a.r, x + h * a.x_head, w0, w1);
                U::store(out + h * a.o_head + t.at0, w0);
                U::store(out + h * a.o_head + t.at1, w1);
            }
        } else {
            const int at = a.r.dims + (u - units) * P;
            for (int h = in / (units + rest); h < a.heads; h += spread) {
                u32x4_t w0;
                if constexpr (VEC)
                    w0 = *(const u32x4_t *)(x + h * a.x_head + at);
                else
                    w0[0] = x[h * a.x_head + at];
                U::store(out + h * a.o_head + at, w0);
            }
        }
    }
}

struct EnterArgs {
    RowsArgs c;  // the cache; keys and values
    RotaryArgs r;
    const char *q;
    char *q_out;
    int64_t q_row, q_head, o_row, o_head;
    int q_heads, q_sets, q_each;  // sets of so many query heads
};

// Rows into the cache, keys and queries turned on the way: a workgroup per block of
// 32 positions and either one key-value head or a set of query heads, which share
// their angles.  Keys are stored as they come, a piece of 16 bytes each; values
// are turned into their layout through LDS.  Bound by HBM: 10,301 rows of 32/8 heads of
// 128 in bf16 50 us (253 MB read and written, 5.1 TB/s; a copy of 1 GiB 5.2), in fp32 107
// (4.7).  48 rows in fp32 8 us, the latency of the lookups (start, length, page) before
// the rows.
template <int ST, bool VEC>
__global__ __launch_bounds__(256) void enter_kernel(EnterArgs a, int64_t items) {
    using U = Unit<ST, VEC>;
    using T = typename U::T;
    constexpr int E = U::E, P = VEC ? E : 1;
    extern __shared__ __align__(16) char lds_rows[];  // the block's values [32][dim + E]
    const RowsArgs &c = a.c;
    const int dim = c.dim, ld = dim + E, units = a.r.dims / 2 / U::N, rest = (dim - a.r.dims) / P;
    T *rows = (T *)lds_rows;
    const int roles = c.heads + a.q_sets;
    for (int64_t w = blockIdx.x; w < items * roles; w += gridDim.x) {
        const int64_t item = w / roles;
        const int role = (int)(w % roles);
        int64_t b = item, blk = 0, row0 = item, count = 1;  // the sequence's rows
        if (c.starts) {
            auto base = [&](int64_t x) { return ((int64_t)c.starts[x] >> 5) + 2 * x; };
            b = last_at_or_below(c.nseq, item, threadIdx.x & 63, base);
            blk = item - base(b);
            row0 = c.starts[b];
            count = c.starts[b + 1] - row0;
        }
        const int64_t end = c.lens[b], first = end - count;  // positions
        const int64_t p0 = ((first >> 5) + blk) * kKvBlock;
        if (blk < 0 || count <= 0 || p0 >= end) continue;
        // positions t of the block that have a row
        const int64_t from = max(row0 < 0 ? first - row0 : first, p0);
        const int64_t to = min(min(end, first + (c.nrows - row0)), p0 + kKvBlock);
        if (from >= to) continue;
        const int t0 = (int)(from - p0), n = (int)(to - from);
        const int64_t row_at = row0 + (from - first);
        if (role >= c.heads) {
            const int h0 = (role - c.heads) * a.q_each, h1 = min(h0 + a.q_each, a.q_heads);
            for (int x = threadIdx.x; x < n * (units + rest); x += 256) {
                const int t = x / (units + rest), u = x % (units + rest);
                const T *src = (const T *)a.q + (row_at + t) * a.q_row;
                T *dst = (T *)a.q_out + (row_at + t) * a.o_row;
                if (u < units) {
                    U turn;
                    turn.angles(a.r, u, from + t);
                    for (int h = h0; h < h1; ++h) {
                        u32x4_t w0, w1;
                        turn.apply(a.r, src + h * a.q_head, w0, w1);
                        U::store(dst + h * a.o_head + turn.at0, w0);
                        U::store(dst + h * a.o_head + turn.at1, w1);
                    }
                } else {
                    const int at = a.r.dims + (u - units) * P;
                    for (int h = h0; h < h1; ++h) {
                        u32x4_t w0;
                        if constexpr (VEC)
                            w0 = *(const u32x4_t *)(src + h * a.q_head + at);
                        else
                            w0[0] = src[h * a.q_head + at];
                        U::store(dst + h * a.o_head + at, w0);
                    }
                }
            }
            continue;
        }
        if (p0 < 0) continue;
        char *const place = block_of(c, (int)b, p0, sizeof(T));
        if (!place) {
            if (p0 >> c.page_shift >= c.width && threadIdx.x == 0)
                atomicOr(&c.status[0], kStatusWidth);
            continue;
        }
        if (c.status[2] && end <= c.width << c.page_shift) {  // some page may take no new rows
            const int last = c.table[b * c.width + ((end - 1) >> c.page_shift)];
            if ((unsigned)last < (unsigned)c.npages && c.closed[last]) continue;
        }
        T *const kd = (T *)(place + role * c.head_off);
        char *const vd = (char *)kd + c.kv_off;
        const T *ks = (const T *)c.k + role * c.k_head + row_at * c.k_row;
        const T *vs = (const T *)c.v + role * c.v_head + row_at * c.v_row;
        const int pieces = dim / E;
        __syncthreads();  // (the last block's values have been read)
        for (int x = threadIdx.x; x < n * pieces; x += 256) {
            const int t = x / pieces, p = x % pieces;
            *(u32x4_t *)(rows + (t0 + t) * ld + p * E) =
                load_piece<ST>((const char *)(vs + t * c.v_row), p * E, c.v_vec);
        }
        for (int x = threadIdx.x; x < n * (units + rest); x += 256) {
            const int t = x / (units + rest), u = x % (units + rest);
            const T *src = ks + t * c.k_row;
            if (u < units) {
                U turn;
                turn.angles(a.r, u, from + t);
                u32x4_t w0, w1;
                turn.apply(a.r, src, w0, w1);
                U::store(kd + key_place<ST>(t0 + t, turn.at0, dim), w0);
                U::store(kd + key_place<ST>(t0 + t, turn.at1, dim), w1);
            } else {
                const int at = a.r.dims + (u - units) * P;
                u32x4_t w0;
                if constexpr (VEC)
                    w0 = *(const u32x4_t *)(src + at);
                else
                    w0[0] = src[at];
                U::store(kd + key_place<ST>(t0 + t, at, dim), w0);
            }
        }
        __syncthreads();
        store_values<ST>(rows, ld, (T *)vd, dim, t0, t0 + n);
    }
}

// Pieces of 16 bytes, each in one place of the layouts?
bool pieces_fit(const vs_rotary *r, int64_t head_dim, int64_t e) {
    const int64_t E = 16 / e;
    return head_dim % E == 0 && r->dims % (2 * E) == 0;
}

int check_rotary(const vs_rotary *r, int64_t head_dim) {
    if (r->dims > head_dim)
        return report(VS_ERR_INVALID, "rotary of %d dimensions on heads of %lld", r->dims,
                      (long long)head_dim);
    return VS_OK;
}

template <int ST, bool VEC>
hipError_t launch_rotate(const TurnArgs &a, int num_cu, hipStream_t st) {
    // Several heads to a thread where that leaves threads enough.
    using U = Unit<ST, VEC>;
    const int64_t units = a.r.dims / 2 / U::N + (a.copy ? (a.dim - a.r.dims) / (VEC ? U::E : 1) : 0);
    int spread = a.heads;
    while (spread > 1 && a.nrows * units * (spread / 2) >= (int64_t)num_cu * 1024)
        spread = (spread + 1) / 2;
    const int64_t threads = a.nrows * units * spread;
    const dim3 grid((uint32_t)std::max<int64_t>(1, std::min<int64_t>((threads + 255) / 256, 1 << 20)));
    hipLaunchKernelGGL((rotate_kernel<ST, VEC>), grid, dim3(256), 0, st, a, spread);
    return hipGetLastError();
}

}  // namespace
}  // namespace vs

using vs::report;
using vs::report_hip;

extern "C" {

int vs_rotary_create(int device, int64_t dims, const double *radians, float gain, int interleaved,
                     vs_rotary **out) {
    if (!out) return report(VS_ERR_INVALID, "null output handle");
    *out = nullptr;
    if (dims <= 0 || dims % 2) return report(VS_ERR_INVALID, "dims must be even and > 0 (got %lld)", (long long)dims);
    if (dims > 65536) return report(VS_ERR_UNSUPPORTED, "more than 65,536 dimensions");
    if (!radians) return report(VS_ERR_INVALID, "null radians");
    if (!std::isfinite(gain)) return report(VS_ERR_INVALID, "gain is not finite");
    for (int64_t i = 0; i < dims / 2; ++i)
        if (!std::isfinite(radians[i]) || std::fabs(radians[i]) > 0x1p40)
            return report(VS_ERR_INVALID, "radians of pair %lld", (long long)i);
    int rc = vs::check_device(device);
    if (rc) return rc;
    vs::DeviceGuard g(device);
    if (g.err != hipSuccess) return report_hip(g.err, "hipSetDevice");
    vs_rotary *r = new (std::nothrow) vs_rotary();
    uint64_t *turns = new (std::nothrow) uint64_t[dims / 2];
    if (!r || !turns) {
        delete r;
        delete[] turns;
        return report(VS_ERR_OOM, "host allocation");
    }
    for (int64_t i = 0; i < dims / 2; ++i) {
        // Whole turns make no difference, and are taken off in radians first: 2 pi in
        // two parts, of 64 bits each, so that what is left is good to 2^-64 of itself
        // however many they are.
        const long double turn = 0xc90fdaa22168c235p-61L, more = -0xece675d1fc8f8cbbp-127L;
        const long double whole = std::rint((long double)radians[i] / turn);
        long double t = std::fma(-whole, more, std::fma(-whole, turn, (long double)radians[i])) / turn;
        t -= std::floor(t);
        const long double n = std::round(t * 0x1p64L);
        turns[i] = n >= 0x1p64L ? 0 : (uint64_t)n;
    }
    r->device = device;
    r->dims = (int)dims;
    r->interleaved = interleaved != 0;
    r->gain = gain;
    r->num_cu = vs::cu_count(device);
    void *p = nullptr;
    hipError_t e = vs::device_alloc(&p, (size_t)(dims / 2) * sizeof(uint64_t));
    r->turns = (uint64_t *)p;
    if (e == hipSuccess)
        e = hipMemcpy(p, turns, (size_t)(dims / 2) * sizeof(uint64_t), hipMemcpyHostToDevice);
    if (e == hipSuccess) e = hipStreamSynchronize(nullptr);  // (before any stream's call)
    delete[] turns;
    if (e != hipSuccess) {
        if (r->turns) (void)hipFree(r->turns);
        delete r;
        return report_hip(e, "rotary frequencies");
    }
    *out = r;
    return VS_OK;
}

void vs_rotary_destroy(vs_rotary *r) {
    if (!r) return;
    vs::DeviceGuard g(r->device);
    (void)hipDeviceSynchronize();
    if (r->turns) (void)hipFree(r->turns);
    delete r;
}

int vs_rotary_apply(const vs_rotary *r, int dtype, const void *x, int64_t x_row, int64_t x_head,
                    const int32_t *positions, int64_t nrows, int64_t heads, int64_t head_dim,
                    void *out, int64_t out_row, int64_t out_head, int backward, void *stream) {
    if (!r) return report(VS_ERR_INVALID, "null handle");
    if (dtype != VS_DTYPE_F32 && dtype != VS_DTYPE_BF16)
        return report(VS_ERR_INVALID, "unknown dtype code %d", dtype);
    if (nrows < 0 || heads <= 0 || head_dim <= 0)
        return report(VS_ERR_INVALID, "nrows must be >= 0, heads and head_dim > 0");
    if (nrows > INT32_MAX || heads > (1 << 16) || head_dim > 65536)
        return report(VS_ERR_UNSUPPORTED, "more than 2^31 - 1 rows, 65,536 heads or dimensions");
    int rc = vs::check_rotary(r, head_dim);
    if (rc) return rc;
    for (int64_t s : {x_row, x_head, out_row, out_head})
        if (!vs::stride_ok(s, nrows)) return report(VS_ERR_INVALID, "stride %lld", (long long)s);
    if (nrows == 0) return VS_OK;
    const int64_t e = dtype == VS_DTYPE_BF16 ? 2 : 4;
    if (!x || !out || !positions) return report(VS_ERR_INVALID, "null buffer");
    if (((uintptr_t)x | (uintptr_t)out) % e || (uintptr_t)positions % 4)
        return report(VS_ERR_INVALID, "a buffer is not aligned to its elements");
    const bool same =
        x == out && (x_row == out_row || nrows == 1) && (x_head == out_head || heads == 1);
    const vs::Extent from(x, x_row, x_head, nrows, heads, head_dim, e),
        to(out, out_row, out_head, nrows, heads, head_dim, e);
    if (!same && vs::meet(from, to))
        return report(VS_ERR_INVALID, "out overlaps x (in place, it is x with its strides)");
    if (vs::overlap(to.low, to.bytes, positions, nrows * 4))
        return report(VS_ERR_INVALID, "out overlaps positions");
    vs::DeviceGuard g(r->device);
    if (g.err != hipSuccess) return report_hip(g.err, "hipSetDevice");
    vs::TurnArgs a = {};
    a.r = {r->turns, r->gain, r->dims, r->interleaved};
    a.back = backward != 0;
    a.x = (const char *)x;
    a.out = (char *)out;
    a.positions = positions;
    a.x_row = x_row;
    a.x_head = x_head;
    a.o_row = out_row;
    a.o_head = out_head;
    a.nrows = nrows;
    a.heads = (int)heads;
    a.dim = (int)head_dim;
    a.copy = !same && head_dim > r->dims;
    const bool vec = vs::pieces_fit(r, head_dim, e) && vs::pieces_ok(x, x_row, x_head, e) &&
                     vs::pieces_ok(out, out_row, out_head, e);
    hipStream_t st = (hipStream_t)stream;
    hipError_t err = e == 2 ? vec ? vs::launch_rotate<1, true>(a, r->num_cu, st)
                                  : vs::launch_rotate<1, false>(a, r->num_cu, st)
                     : vec ? vs::launch_rotate<0, true>(a, r->num_cu, st)
                           : vs::launch_rotate<0, false>(a, r->num_cu, st);
    return err == hipSuccess ? VS_OK : report_hip(err, "rotary");
}

int vs_kv_append_rotary(vs_kv *kv, const vs_kv_seqs *s, int64_t layer, const vs_rotary *r,
                        const void *k, int64_t k_row, int64_t k_head, const void *v, int64_t v_row,
                        int64_t v_head, const void *q, int64_t q_row, int64_t q_head, int64_t heads,
                        void *q_out, int64_t out_row, int64_t out_head, const int32_t *starts,
                        int64_t nrows, void *stream) {
    if (!kv || !r) return report(VS_ERR_INVALID, "null handle");
    int rc = vs::check_seqs(kv, s);
    if (rc) return rc;
    vs::EnterArgs a = {};
    rc = vs::fill_rows(kv, s, layer, a.c);
    if (!rc) rc = vs::check_rotary(r, kv->head_dim);
    if (rc) return rc;
    if (r->device != kv->device)
        return report(VS_ERR_INVALID, "rotary on device %d, the cache on %d", r->device, kv->device);
    if (nrows < 0 || (!starts && nrows != s->nseq))
        return report(VS_ERR_INVALID, "nrows %lld: without starts, one row per sequence",
                      (long long)nrows);
    if (nrows > INT32_MAX) return report(VS_ERR_UNSUPPORTED, "more than 2^31 - 1 rows");
    if (!q != !q_out) return report(VS_ERR_INVALID, "q and q_out are given together or not at all");
    if (q && (heads <= 0 || heads > (1 << 16)))
        return report(VS_ERR_INVALID, "heads %lld out of range [1, 65,536]", (long long)heads);
    for (int64_t x : {k_row, k_head, v_row, v_head, q_row, q_head, out_row, out_head})
        if (!vs::stride_ok(x, nrows)) return report(VS_ERR_INVALID, "stride %lld", (long long)x);
    if (nrows == 0 || s->nseq == 0) return VS_OK;
    if (!k || !v) return report(VS_ERR_INVALID, "null k or v");
    const int64_t e = vs::kv_elem(kv->dtype), d = kv->head_dim, hk = kv->kv_heads;
    if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)q | (uintptr_t)q_out) % e || (uintptr_t)starts % 4)
        return report(VS_ERR_INVALID, "a buffer is not aligned to its elements");
    if (q) {
        const bool same = q == q_out && (q_row == out_row || nrows == 1) &&
                          (q_head == out_head || heads == 1);
        const vs::Extent to(q_out, out_row, out_head, nrows, heads, d, e);
        if (!same && vs::meet(vs::Extent(q, q_row, q_head, nrows, heads, d, e), to))
            return report(VS_ERR_INVALID, "q_out overlaps q (in place, it is q with its strides)");
        if (vs::meet(vs::Extent(k, k_row, k_head, nrows, hk, d, e), to) ||
            vs::meet(vs::Extent(v, v_row, v_head, nrows, hk, d, e), to))
            return report(VS_ERR_INVALID, "q_out overlaps k or v");
        if (vs::over_places(to, s, starts))
            return report(VS_ERR_INVALID, "q_out overlaps starts, lens or table");
        a.q_heads = (int)heads;
    }
    vs::DeviceGuard g(kv->device);
    if (g.err != hipSuccess) return report_hip(g.err, "hipSetDevice");
    a.r = {r->turns, r->gain, r->dims, r->interleaved};
    a.c.starts = starts;
    a.c.nrows = nrows;
    a.c.k = (const char *)k;
    a.c.v = (const char *)v;
    a.c.k_row = k_row;
    a.c.k_head = k_head;
    a.c.v_row = v_row;
    a.c.v_head = v_head;
    a.c.v_vec = vs::pieces_ok(v, v_row, v_head, e);
    a.q = (const char *)q;
    a.q_out = (char *)q_out;
    a.q_row = q_row;
    a.q_head = q_head;
    a.o_row = out_row;
    a.o_head = out_head;
    const int64_t items = starts ? nrows / vs::kKvBlock + 2 * s->nseq + 1 : nrows;
    // A set of four query heads moves as much as a key-value head; fewer where the
    // call is small.
    a.q_each = items * (hk + a.q_heads / 4) >= 2 * kv->num_cu ? 4 : 1;
    a.q_sets = (a.q_heads + a.q_each - 1) / a.q_each;
    const bool vec = vs::pieces_fit(r, d, e) && vs::pieces_ok(k, k_row, k_head, e) &&
                     (!q || (vs::pieces_ok(q, q_row, q_head, e) && vs::pieces_ok(q_out, out_row, out_head, e)));
    const dim3 grid((uint32_t)std::min<int64_t>(items * (hk + a.q_sets), 1 << 20));
    const size_t lds = (size_t)vs::kKvBlock * (d * e + 16);
    hipStream_t st = (hipStream_t)stream;
    if (e == 2 && vec)
        hipLaunchKernelGGL((vs::enter_kernel<1, true>), grid, dim3(256), lds, st, a, items);
    else if (e == 2)
        hipLaunchKernelGGL((vs::enter_kernel<1, false>), grid, dim3(256), lds, st, a, items);
    else if (vec)
        hipLaunchKernelGGL((vs::enter_kernel<0, true>), grid, dim3(256), lds, st, a, items);
    else
        hipLaunchKernelGGL((vs::enter_kernel<0, false>), grid, dim3(256), lds, st, a, items);
    hipError_t err = hipGetLastError();
    return err == hipSuccess ? VS_OK : report_hip(err, "append");
}

}  // extern "C"

// vs_logits.h -- rows of logits in a wave's registers, and lists of the largest of
// them, shared by beam search and the log probabilities of given tokens.
#pragma once

#include "vs_device.h"
#include "vs_host.h"
#include "vs_wave.h"

struct vs_beam {
    int device = 0;
    int num_cu = 256;
    vs::StreamScratch scratch;
};

#define VS_NINF (-__builtin_huge_valf())

namespace vs {

constexpr int kMaxK = 64;
constexpr int kLongStep = 32;       // logits per lane and step, in large calls
constexpr int kShortStep = 16;      // and small ones
constexpr int kCap = 256;           // candidates per piece kept in LDS
constexpr float kLog2e = 1.44269504088896340736f;

// Larger float, larger code; both zeros have one code.
__device__ __forceinline__ uint32_t code_of(float x) {
    const uint32_t u = bits_of(x + 0.f);  // (-0 + 0 is 0)
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t c) {
    return float_of(c & 0x80000000u ? c & 0x7FFFFFFFu : ~c);
}

// The larger of three, passing quiet NaNs over (fmaxf would first quiet each of
// its operands, an instruction more per logit; a signalling NaN may get
// through, and the row's sum is a NaN then in any case).
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// 64 PER consecutive logits of a row in a wave's registers.  Which lane holds
// which token goes by the token alone, wherever the row starts: equal rows have
// equal sums to the bit, and their beams tie.
template <int ST, int PER>
struct Step {
    static constexpr int E = ST ? 8 : 4, NL = PER / E, ES = 16 / E;
    u32x4_t w[NL];

    // (unaligned 16-byte loads: rows start anywhere)
    __device__ __forceinline__ void load(const char *row, int first, int vocab, int lane) {
        const int left = vocab - first;
#pragma unroll
        for (int l = 0; l < NL; ++l) {
            if ((l + 1) * 64 * E <= left) {
                __builtin_memcpy(&w[l], row + (int64_t)(first + (l * 64 + lane) * E) * ES, 16);
            } else if (l * 64 * E >= left) {
                w[l] = ST ? u32x4_t{0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u}
                          : u32x4_t{0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u};
            } else {
                // where the row ends: one load per token, all in flight
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = first + (l * 64 + lane) * E + i * (E / 4);
                    if constexpr (ST) {
                        const uint16_t *p = (const uint16_t *)row;
                        const uint32_t lo = p[min(t, vocab - 1)], hi = p[min(t + 1, vocab - 1)];
                        w[l][i] = (t < vocab ? lo : 0xFF80u) | (t + 1 < vocab ? hi : 0xFF80u) << 16;
                    } else {
                        const uint32_t v = ((const uint32_t *)row)[min(t, vocab - 1)];
                        w[l][i] = t < vocab ? v : 0xFF800000u;
                    }
                }
            }
        }
    }
    __device__ __forceinline__ float value(int i) const {
        if constexpr (ST) {
            const uint32_t x = w[i / E][i % E / 2];
            return float_of(i % 2 ? x & 0xFFFF0000u : x << 16);
        } else {
            return float_of(w[i / E][i % E]);
        }
    }
    static __device__ __forceinline__ int token(int first, int i, int lane) {
        return first + ((i / E) * 64 + lane) * E + i % E;
    }
    // the logit of token(first, i, lane), from memory
    static __device__ __forceinline__ float reload(const char *row, int first, int i, int vocab,
                                                   int lane) {
        const int t = token(first, i, lane);
        if (t >= vocab) return VS_NINF;
        return ST ? float_of((uint32_t)((const uint16_t *)row)[t] << 16) : ((const float *)row)[t];
    }
};

// How many of the lanes in `in` come before this one.
__device__ __forceinline__ int below(uint64_t in) {
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32),
                                          __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0));
}

// Larger logit first, then the lower token, as one 64-bit number.
__device__ __forceinline__ uint64_t key_of(float v, int token) {
    return (uint64_t)code_of(v) << 32 | ~(uint32_t)token;
}

// The wave's list of n keys (at most kCap) cut to its k best, in order.
__device__ __forceinline__ void cut_list(uint64_t *cand, int n, int k, int lane) {
    uint64_t me[kCap / 64];
    int rank[kCap / 64];
    lds_wave_sync();
#pragma unroll
    for (int c = 0; c < kCap / 64; ++c) {
        me[c] = c * 64 + lane < n ? cand[c * 64 + lane] : 0;
        rank[c] = c * 64 + lane < n ? 0 : k;
    }
    for (int j = 0; j < n; ++j) {
        const uint64_t o = cand[j];
#pragma unroll
        for (int c = 0; c < kCap / 64; ++c) rank[c] += o > me[c];
    }
    lds_wave_sync();
#pragma unroll
    for (int c = 0; c < kCap / 64; ++c)
        if (rank[c] < k) cand[rank[c]] = me[c];
    lds_wave_sync();
}

}  // namespace vs

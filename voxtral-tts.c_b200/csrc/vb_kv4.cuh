/*
 * vb_kv4.cuh - what the kernels of attention over the 4-bit cache share (vb_kv4_attn.cu, vb_kv4_prompt.cu).
 */
#ifndef VB_KV4_CUH
#define VB_KV4_CUH

#include <limits.h>
#include <type_traits>

#include "vb_serve.cuh"

namespace vb {

/* One of 32, 64, 96, 128, 192, 256 values a head, as a constant */
#define VB_KV4_DIMS(blocks, call) \
    switch (blocks) {             \
    case 1: return call(1);       \
    case 2: return call(2);       \
    case 3: return call(3);       \
    case 4: return call(4);       \
    case 6: return call(6);       \
    default: return call(8);      \
    }

/* Weights are taken against a reference that trails the largest by at most 2^2 and held times 2^13, so that the largest are 2^15 and FP16's smallest
 * step, 2^-24, is 2^-37 of the reference. (2^8 and 2^7 need fewer changes of the reference, and lost a tenth of weights of 2^-29; level
 * in time with a few rows.) */
constexpr float kKv4Trail = 2.0f, kKv4Bias = 13.0f;
constexpr int kKv4Rest = 8;                   /* sums and results of a part leave the accumulators times 2^-8: */
constexpr float kKv4Out = 0x1p-21f;           /* 2^-13 2^-8, sums */
constexpr int kKv4Down = 127 + 13 + 21;       /* and results, of values based on a scale byte times 2^13 */
/* FP16 terms of a weight */
template <class T>
constexpr int kWeightTerms = std::is_same<T, __nv_bfloat16>::value ? 1 : 2;

struct Kv4Attn {
    Kv4 c;
    const int *lengths, *rows;
    int max_rows, heads, group, row_tiles, split, wide, wide_out;
    int tail0, tail_units, tail_parts;       /* of vb_kv4_prompt.cu */
    float scale;
    float *lse;
    const float *mass_in;
    float *mass_out;
    float *part, *aside;
    unsigned *tickets, *rooms;
    int n_rooms;
    int *status;
};

VB_DEVINL uint32_t half_mul(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
VB_DEVINL uint32_t half_pack(float a, float b) { return serve_pack(a, b, (const __half *)nullptr); }
VB_DEVINL float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

/* N bytes side by side (aligned to N's largest power of two) */
template <int N>
VB_DEVINL void get_bytes(const uint8_t *p, uint32_t (&b)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const uint32_t w = reinterpret_cast<const uint32_t *>(p)[i];
#pragma unroll
            for (int j = 0; j < 4; j++) b[4 * i + j] = (w >> (8 * j)) & 255u;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            const uint32_t w = reinterpret_cast<const uint16_t *>(p)[i];
            b[2 * i] = w & 255u;
            b[2 * i + 1] = w >> 8;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) b[i] = p[i];
    }
}
/* N scale bytes side by side as numbers (infinity for 255: its block is zeros, so that it adds NaN). A shift to the left goes to the
 * pipe of the multiply-adds, which has room */
template <int N>
VB_DEVINL void get_scales(const uint8_t *p, float (&f)[N]) {
    constexpr int kEach = N % 4 == 0 ? 4 : N % 2 == 0 ? 2 : 1;
#pragma unroll
    for (int i = 0; i < N / kEach; i++) {
        const uint32_t w = kEach == 4 ? reinterpret_cast<const uint32_t *>(p)[i] : kEach == 2 ? reinterpret_cast<const uint16_t *>(p)[i] : p[i];
#pragma unroll
        for (int j = 0; j < kEach; j++) f[kEach * i + j] = __uint_as_float((j < 3 ? w << (23 - 8 * j) : w >> 1) & 0x7f800000u);
    }
}
/* N words side by side (aligned to N's largest power of two, up to four) */
template <int N>
VB_DEVINL void get_words(const uint8_t *p, uint32_t (&w)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const uint4 v = reinterpret_cast<const uint4 *>(p)[i];
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            const uint2 v = reinterpret_cast<const uint2 *>(p)[i];
            w[2 * i] = v.x; w[2 * i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) w[i] = reinterpret_cast<const uint32_t *>(p)[i];
    }
}
/* Which (sequence, unit, split) a CTA has. A unit is PAIRS (row, query head) pairs of a KV head, a share a number of tiles of TOKENS. Where
 * there are fewer units than CTAs that run at once (a.split), sequences are cut so that all CTAs have about the same number of tiles, by
 * their actual lengths: the smallest share, in whole rounds and `least` at least, with which there are enough CTAs. (With as many
 * splits for each sequence, four of 65536 to 131072 tokens took the time of four of 131072.) Otherwise every unit has a CTA. `round` is a
 * power of two. */
struct Kv4Place {
    int seq, unit, split, share;
};
template <int PAIRS, int TOKENS>
VB_DEVINL Kv4Place kv4_place(const Kv4Attn &a, int round, int least, int most_splits) {
    if (!a.split) {
        const int units = a.row_tiles * a.c.kv_heads;
        return {(int)blockIdx.x / units, (int)blockIdx.x % units, 0, INT_MAX};
    }
    const int lane = threadIdx.x & 31, n_cta = gridDim.x;
    auto tiles_of = [&](int s, int *units) {
        const Kv4Span span = kv4_span(a.lengths, a.rows, a.max_rows, s, a.c.capacity);
        *units = (span.rows * a.group + PAIRS - 1) / PAIRS * a.c.kv_heads;
        return (span.length + TOKENS - 1) / TOKENS;
    };
    /* the first 32 sequences stay in registers; there are at most a few hundred, or every unit has a CTA of its own */
    int units0 = 0;
    const int tiles0 = lane < a.c.seqs ? tiles_of(lane, &units0) : 0;
    int most = tiles0;
    float work = (float)max(tiles0, 1) * (float)units0;
    for (int s = lane + 32; s < a.c.seqs; s += 32) {
        int units;
        const int tiles = tiles_of(s, &units);
        most = max(most, tiles);
        work += (float)max(tiles, 1) * (float)units;
    }
    most = __reduce_max_sync(0xffffffffu, most);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) work += __shfl_xor_sync(0xffffffffu, work, o);
    /* a quotient to within one: no more is asked of it, but to be the same for every CTA */
    auto quotient = [](int x, int by) { return (int)__fdividef((float)x, (float)by); };
    int share = max((int)__fdividef(work, (float)n_cta), quotient(most, most_splits)) + 1;
    share = max(least, (share + round - 1) & -round);
    /* a unit's last part may be short: a little more, in steps of a sixteenth, until the CTAs are enough */
    while (share < most) {
        unsigned n = units0 * (unsigned)max(1, (tiles0 + share - 1) / share);
        for (int s = lane + 32; s < a.c.seqs; s += 32) {
            int units;
            const int tiles = tiles_of(s, &units);
            n += units * (unsigned)max(1, (tiles + share - 1) / share);
        }
        if ((int)__reduce_add_sync(0xffffffffu, n) <= n_cta && (most + share - 1) / share <= most_splits) break;
        share += max(round, (share >> 4) & -round);
    }
    /* this CTA's place: sequence by sequence, all units' first parts, then their second ones */
    int left = blockIdx.x;
    for (int s0 = 0; s0 < a.c.seqs; s0 += 32) {
        int units = units0, tiles = tiles0;
        if (s0 > 0) tiles = s0 + lane < a.c.seqs ? tiles_of(s0 + lane, &units) : 0;
        if (s0 + lane >= a.c.seqs) units = 0;
        const int mine = units * max(1, (tiles + share - 1) / share);
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const unsigned there = __ballot_sync(0xffffffffu, left < upto);
        if (there) {
            const int who = __ffs(there) - 1;
            const int at = left - (__shfl_sync(0xffffffffu, upto, who) - __shfl_sync(0xffffffffu, mine, who)), n = __shfl_sync(0xffffffffu, units, who);
            return {s0 + who, at % n, at / n, share};
        }
        left -= __shfl_sync(0xffffffffu, upto, 31);
    }
    return {a.c.seqs, 0, 0, share};
}

/* ------------------------------------------------------------------ scales too far apart
 * The tensor cores take values as FP16, based on the largest scale: exact where scales lie within 2^36 of one another. A CTA that meets others
 * (kv4_far; scales that have risen by more than kKv4Rise: what a row has of smaller ones fell with them) works its part out again here, in fp32 and
 * with bases of a row's own, so that what a row does not see does not reach it and a large value that weighs little leaves the others as they are. A
 * function of its own: inlined into vb_kv4_attn.cu's loop for a tile at a time it cost every call 5 % (four sequences of 131072 tokens
 * 98 -> 104 us). One row over 4208 tokens 14 us -> 126, over 131072 133 -> 4960, 1203 fp32 rows 0.2 ms -> 19. */
constexpr int kKv4Rise = 64;

/* 2^e, |e| up to 252, as a product of two */
VB_DEVINL float2 kv4_power(int e) { return make_float2(__uint_as_float((uint32_t)(127 + (e >> 1)) << 23), __uint_as_float((uint32_t)(127 + e - (e >> 1)) << 23)); }

/* A head's planes */
struct Kv4Head {
    const uint8_t *k, *v, *ks, *vs;
};
template <int NB>
VB_DEVINL Kv4Head kv4_head(const Kv4 &c, size_t row0) { return {c.k + row0 * (NB * 16), c.v + row0 * (NB * 16), c.ks + row0 * NB, c.vs + row0 * NB}; }

/* A query row into q_s, by a warp, the largest brought to [2^14, 2^15) as on the tensor cores: no product of finite numbers passes fp32. Returns what
 * its scores are to be multiplied by to be powers of two. */
template <int NB, class T>
VB_DEVINL float kv4_plain_query(const T *q, float scale, float *q_s) {
    const int lane = threadIdx.x & 31;
    uint32_t most = 0;
    for (int d = lane; d < NB * 32; d += 32) most = max(most, __float_as_uint(serve_get(q + d)) & 0x7fffffffu);
    most = __reduce_max_sync(0xffffffffu, most);
    const uint32_t e = most >> 23, field = e == 0u || e == 255u ? 127u : min(268u - e, 253u);
    __syncwarp();
    for (int d = lane; d < NB * 32; d += 32) q_s[d] = serve_get(q + d) * __uint_as_float(field << 23);
    __syncwarp();
    return scale * 1.44269504f * __uint_as_float((254u - field) << 23);
}
/* Its score with a row of the cache, by a lane. */
template <int NB>
VB_DEVINL float kv4_plain_score(const Kv4Head &c, size_t row, const float *q_s, float mul) {
    float sums[NB], s = 0.0f;
#pragma unroll
    for (int b = 0; b < NB; b++) sums[b] = 0.0f;
#pragma unroll 1
    for (int t = 0; t < 4; t++) {
        uint32_t w[NB];
        get_words<NB>(c.k + row * (NB * 16) + t * (NB * 4), w);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            uint32_t h[4];
            kv4_halves(w[b], h);
            const float4 x = *reinterpret_cast<const float4 *>(q_s + 32 * b + 8 * t), y = *reinterpret_cast<const float4 *>(q_s + 32 * b + 8 * t + 4);
            const float2 k0 = kv4_f2(h[0]), k1 = kv4_f2(h[1]), k2 = kv4_f2(h[2]), k3 = kv4_f2(h[3]);
            sums[b] = fmaf(k0.x, x.x, fmaf(k0.y, x.y, fmaf(k1.x, x.z, fmaf(k1.y, x.w, sums[b]))));
            sums[b] = fmaf(k2.x, y.x, fmaf(k2.y, y.y, fmaf(k3.x, y.z, fmaf(k3.y, y.w, sums[b]))));
        }
    }
#pragma unroll
    for (int b = 0; b < NB; b++) {
        const uint32_t byte = c.ks[row * NB + b];
        const float2 f = kv4_power((int)min(byte, 252u) - 127);
        s += byte == 255u ? __uint_as_float(0x7fffffffu) : sums[b] == 0.0f ? 0.0f : sums[b] * f.x * mul * f.y;
    }
    return s;
}
/* A query row over the rows tok0 .. tok1 of a head, by a warp: its reference and sum; results [NB * 32] in out_s. q_s has room for a row. (The head by
 * value: a reference to a kernel's arguments has all of them copied to the stack first.) */
template <int NB, class T>
__device__ __noinline__ float2 kv4_plain_row(Kv4Head c, const T *q, float scale, int tok0, int tok1, float *q_s, float *out_s) {
    const int lane = threadIdx.x & 31;
    const float mul = kv4_plain_query<NB>(q, scale, q_s);
    float ref = -INFINITY, sum = 0.0f, o[NB];
    int base[NB];
    uint32_t nan = 0;
#pragma unroll
    for (int i = 0; i < NB; i++) o[i] = 0.0f, base[i] = 0;
    for (int j0 = tok0; j0 < tok1; j0 += 32) {
        /* scores: a lane a token */
        const int j = j0 + lane, n = min(32, tok1 - j0);
        const size_t row = min(j, tok1 - 1);
        float s = kv4_plain_score<NB>(c, row, q_s, mul);
        if (j >= tok1) s = -INFINITY;
        float top = s;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float now = fmaxf(ref, top), fall = ref > -INFINITY ? exp2_fast(ref - now) : 0.0f;
        ref = now;
        const float p = j >= tok1 ? 0.0f : exp2_fast(s - (ref > -INFINITY ? ref : 0.0f));
        float all = p;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) all += __shfl_xor_sync(0xffffffffu, all, x);
        sum = fmaf(sum, fall, all);
        /* values: a lane one of every block */
#pragma unroll
        for (int i = 0; i < NB; i++) {
            const uint32_t byte = j < tok1 ? c.vs[row * NB + i] : 0u;
            if (__any_sync(0xffffffffu, byte == 255u)) nan |= 1u << i;
            const int rise = max(0, (int)__reduce_max_sync(0xffffffffu, byte == 255u ? 0u : byte) - base[i]);
            base[i] += rise;
            o[i] *= rise > 126 ? 0.0f : fall * __uint_as_float((uint32_t)(127 - rise) << 23);
            /* a lane's own token: its weight times its scale against the base */
            const float2 f = kv4_power(byte == 255u ? 0 : min((int)byte - base[i], 0));
            const float weight = p * f.x * f.y;
            const uint8_t *values = c.v + (size_t)j0 * (NB * 16) + kv4_value_half(8 * i + (lane >> 2), NB) * 2 + ((lane & 3) >> 1);
            float part = 0.0f;
#pragma unroll 2
            for (int x0 = 0; x0 < n; x0 += 4) {        /* what is behind the last token weighs nothing; four conversions of a word together (one byte
                                                        * of a word alone, in an unrolled loop, came out as zeros) */
                uint32_t four = 0, h[4];
#pragma unroll
                for (int x = 0; x < 4; x++) four |= (uint32_t)values[(size_t)min(x0 + x, n - 1) * (NB * 16)] << (8 * x);
                kv4_halves(four, h);
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const float2 pair = kv4_f2(h[x]);
                    part = fmaf(lane & 1 ? pair.y : pair.x, __shfl_sync(0xffffffffu, weight, x0 + x), part);
                }
            }
            o[i] += part;
        }
    }
#pragma unroll
    for (int i = 0; i < NB; i++) {
        const float2 f = kv4_power(base[i] - 127 - kKv4Rest);
        out_s[32 * i + lane] = nan >> i & 1 ? __uint_as_float(0x7fffffffu) : o[i] * f.x * f.y;
    }
    __syncwarp();
    return make_float2(ref, sum * (1.0f / (1 << kKv4Rest)));
}

/* Many rows, heads up to 128 (vb_kv4_prompt.cu) */
template <class T>
int kv4_prompt(const Kv4Attn &a, const ServeRows<T> &q, const ServeRows<T> &out, int sm_count, cudaStream_t st);
template <class T>
int kv4_mass_many(const Kv4Attn &a, const ServeRows<T> &q, cudaStream_t st);
int kv4_prompt_load(int blocks);
/* floats of partial results that it needs */
size_t kv4_prompt_floats(int blocks, int sm_count);
size_t kv4_aside_floats(int blocks, int sm_count);       /* and of sums put aside */

} // namespace vb

#endif

/*
 * vb_kv4_attn.cu - softmax attention over the 4-bit cache, and the weight that each of its tokens was given.
 *
 *   s_ij = scale q_i . k_j,  out_i = sum_j exp(s_ij - lse_i) v_j,  mass_j = sum_i exp(s_ij - lse_i)
 *
 * The codes are exact in FP16, so the products run on FP16 warp-level MMAs (m16n8k16), tokens along M, eight
 * (row, query head) pairs of a KV head along N:
 *   S^T [16 tokens x 8] += K Q^T    a block of 32 at a time, whose sum is multiplied by the token's scale in fp32
 *   O^T [16 dims x 8]   += V^T P^T  values times 2^(e - E + 13), E the largest scale of the block column so far: exact in FP16 where no
 *                                   token's scale is under 2^-36 of the largest; a CTA that meets one works in fp32 (kv4_plain_row)
 * Queries are brought to [2^14, 2^15) by a power of two a row (exact), then one FP16 term (bf16, fp16: exact down to 2^-29
 * of a row's largest) or two (fp32: 22 bits and a sign, down to 2^-39 of the largest). Weights are taken against a running reference that
 * trails the maximum by at most 2^2, times 2^13, so that FP16 holds them from 2^15 down in steps of 2^-24: one term for bf16 results (11 bits against
 * the 8 of the result, 2^-38 of the largest weight at least), two otherwise (22 bits down to 2^-15 of the largest, below that to within 2^-38 of it).
 *
 * A warp walks tiles of 32 tokens with a maximum, sums and accumulators of its own, through a ring of its own that bulk copies
 * fill: no barrier between warps until the end. A sequence's tokens are split over CTAs where there are few of them; the CTA that
 * comes last at a ticket joins the parts.
 *
 * Where tokens are many nothing is saturated: a warp's tile is 607 instructions, of which 283, conversions and integer operations, go to a pipe of half
 * the rate; that pipe is 58 % busy, the issue slots 61, the tensor pipe 26, memory at 63 % of a plain copy's rate. Four warps a scheduler with
 * chains of dependent instructions leave the rest. One row of 32 heads over four sequences of 65536 to 131072 tokens and 8 KV heads of 128, bf16:
 * 104 us, 4.1 TB/s of codes and scales. Over 301 tokens 7.2 us: latencies that wait for one another. Several groups of eight pairs of a KV head
 * each decode its keys and values again: 32 rows and heads of it over 65536 tokens 70 us.
 */
#include <algorithm>
#include <limits.h>

#include "vb_kv4.cuh"
#include "vb_tc.cuh"

namespace vb {

namespace {

constexpr int kAWarps = 8, kAThreads = 32 * kAWarps, kACols = 8, kAKeys = 32;
constexpr int kAStatus = 61;
constexpr int kAMaxSplits = 64;               /* a CTA joins them */

template <int NB>
struct ACfg {
    static constexpr int kDim = NB * 32;
    static constexpr int kCodes = kAKeys * NB * 16, kScales = kAKeys * NB;      /* bytes of a tile's plane */
    static constexpr int kStage = 2 * (kCodes + kScales);
    static constexpr int kStages = NB <= 4 ? 3 : 2;
    static constexpr int kRing = kAWarps * kStages * kStage;
    static constexpr int kMerge = kAWarps * kACols * (kDim + 2) * 4;
    static constexpr int kBig = kRing > kMerge ? kRing : kMerge;
    static constexpr bool kWhole = kv4_whole(NB);
    static constexpr int kVScales = kWhole ? 1 : NB;                            /* scales of a lane's part of a value row */
};

VB_DEVINL void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y));
}
/* without what was there before */
VB_DEVINL void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y), "f"(0.0f));
}
VB_DEVINL uint32_t mat_turn(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
/* A lane's part of a value row, 2 NB bytes, as words (the last one's upper half zero where NB is odd) */
template <int NB>
VB_DEVINL void get_values(const uint8_t *p, uint32_t (&w)[(NB + 1) / 2]) {
    if constexpr (NB % 2 == 0) {
        get_words<NB / 2>(p, w);
    } else {
        const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
        for (int i = 0; i < NB / 2; i++) w[i] = h[2 * i] | ((uint32_t)h[2 * i + 1] << 16);
        w[NB / 2] = h[NB - 1];
    }
}

/* Eight (row, head) pairs are the B operand of K Q^T, in q_s [block][half][term][lane]: column n by warp n, four values a lane. (All of
 * them by one warp: 3450 clocks until they were there, with fp32 heads of 128.) What S is to be multiplied by to be a power of two goes into
 * mul_s. Loads first, so that other things can be begun while they are on their way. */
template <int NB, class T>
struct QueryColumn {
    static constexpr int kGroups = NB * 8, kEach = (kGroups + 31) / 32;
    ServeRaw4<T> raw[kEach];
    VB_DEVINL void load(const ServeRows<T> &q, const Kv4Attn &a, int seq, int kv_head, int pair, int pairs) {
        const int lane = threadIdx.x & 31;
        const bool real = pair < pairs;
        const int row = real ? pair / a.group : 0, head = kv_head * a.group + (real ? pair - row * a.group : 0);
        const T *p = q.data + seq * q.seq + row * q.row + head * q.head;
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            const int at = lane + 32 * i;
            raw[i].none();
            if (real && at < kGroups) raw[i].load(p + at * 4, a.wide);
        }
    }
    template <int QT>
    VB_DEVINL void put(const Kv4Attn &a, int n, uint2 *q_s, float *mul_s) {
        const int lane = threadIdx.x & 31;
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            const float4 x = raw[i].get();
            most = max(max(most, __float_as_uint(x.x) & 0x7fffffffu), __float_as_uint(x.y) & 0x7fffffffu);
            most = max(max(most, __float_as_uint(x.z) & 0x7fffffffu), __float_as_uint(x.w) & 0x7fffffffu);
        }
        most = __reduce_max_sync(0xffffffffu, most);
        /* the largest to [2^14, 2^15); rows of zeros, or with a value that is not finite, as they are */
        const uint32_t e = most >> 23, field = e == 0u || e == 255u ? 127u : min(268u - e, 253u);
        const float down = __uint_as_float((254u - field) << 23);
        float up = __uint_as_float(field << 23);
        if (a.scale <= 0.0f) up = a.scale < 0.0f ? -up : 0.0f;       /* the factor is positive: the largest score is the largest product */
        if (lane == 0) mul_s[n] = fmaxf((a.scale != 0.0f ? fabsf(a.scale) * 1.44269504f : 1.0f) * down, 0x1p-149f);      /* not 0: what is masked stays -inf */
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            const int at = lane + 32 * i;                             /* 8 blocks + 2 t + half */
            if (at >= kGroups) continue;
            uint2 *to = q_s + (((at >> 3) * 2 + (at & 1)) * QT) * 32 + n * 4 + ((at >> 1) & 3);
            const float4 x = raw[i].get();
            const float y[4] = {x.x * up, x.y * up, x.z * up, x.w * up};
            const uint2 w = make_uint2(half_pack(y[0], y[1]), half_pack(y[2], y[3]));
            to[0] = w;
            if constexpr (QT == 2) {
                const float2 f = kv4_f2(w.x), g = kv4_f2(w.y);
                to[32] = make_uint2(half_pack(y[0] - f.x, y[1] - f.y), half_pack(y[2] - g.x, y[3] - g.y));
            }
        }
    }
};

/* Scores of 16 tokens: `at` words of the lane's two tokens (g and g + 8 of them), c: tokens g, g + 8 x columns 2 t, 2 t + 1. */
template <bool FIRST, int QT>
VB_DEVINL void block_scores(float (&s)[4], const uint32_t wa, const uint32_t wb, float fa, float fb, const uint2 (&q)[2][QT]) {
    uint32_t ra[4], rb[4];
    kv4_halves(wa, ra);
    kv4_halves(wb, rb);
    float c[4];
    mma_f16_first(c, ra[0], rb[0], ra[1], rb[1], q[0][0]);
    if constexpr (QT == 2) mma_f16(c, ra[0], rb[0], ra[1], rb[1], q[0][1]);
#pragma unroll
    for (int u = 0; u < QT; u++) mma_f16(c, ra[2], rb[2], ra[3], rb[3], q[1][u]);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float f = j < 2 ? fa : fb;
        s[j] = FIRST ? c[j] * f : fmaf(c[j], f, s[j]);
    }
}

/* grid = CTAs that run at once, or (a.split == 0) sequences x units */
template <int NB, int PT, class T>
__global__ void __launch_bounds__(kAThreads, NB <= 4 ? 2 : 1) kv4_attn_kernel(const Kv4Attn a, const ServeRows<T> q, const ServeRows<T> out) {
    using Cfg = ACfg<NB>;
    constexpr int QT = sizeof(T) == 4 ? 2 : 1, kDim = Cfg::kDim, kW = (NB + 1) / 2, kVS = Cfg::kVScales;
    /* An MMA rounds its sum towards zero: products of 16 tokens by themselves, added up rounded to nearest (112 fp32 pairs of 192 over 34225
     * tokens: 4.7e-7 off 64 bits, 601 us; 5.4e-6 and 581 in one sum, elementary operations 2.8e-6). bf16 results are rounded to far less. */
    constexpr bool kExact = PT == 2;
    extern __shared__ __align__(128) unsigned char a_smem[];
    __shared__ __align__(8) uint64_t full[kAWarps][Cfg::kStages];
    __shared__ __align__(16) uint2 q_s[NB * 2 * QT * 32];
    __shared__ float mul_s[kACols];
    __shared__ int abort_flag, is_last;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    pdl_wait();
    pdl_launch_dependents();       /* after the wait: the masses' kernel reads what this one has waited for */
    const Kv4Place place = kv4_place<kACols, kAKeys>(a, kAWarps, 2 * kAWarps, kAMaxSplits);
    if (place.seq >= a.c.seqs) return;
    const int seq = place.seq, tile_r = place.unit / a.c.kv_heads, kv_head = place.unit - tile_r * a.c.kv_heads, split = place.split, share = place.share;
    QueryColumn<NB, T> column;
    column.load(q, a, seq, kv_head, tile_r * kACols + warp, a.max_rows * a.group);
    const Kv4Span span = kv4_span(a.lengths, a.rows, a.max_rows, seq, a.c.capacity);
    const int pairs = span.rows * a.group, pair0 = tile_r * kACols;
    if (pair0 >= pairs) return;
    const int n_pairs = min(kACols, pairs - pair0);
    const int before = span.length - span.rows;                      /* tokens before row 0 */
    /* tokens that the tile's last row sees, in tiles */
    const int seen = max(0, before + (pair0 + n_pairs - 1) / a.group + 1);
    const int tiles = (seen + kAKeys - 1) / kAKeys;
    const int used = tiles <= share ? 1 : (tiles + share - 1) / share;
    if (split >= used) return;
    const int t_begin = split * share + warp, t_end = used == 1 ? tiles : min(tiles, (split + 1) * share);

    unsigned char *ring = a_smem + warp * Cfg::kStages * Cfg::kStage;
    const size_t row0 = a.c.row(seq, kv_head, 0);
    auto fetch = [&](int tile, int stage) {
        unsigned char *to = ring + stage * Cfg::kStage;
        const size_t row = row0 + (size_t)tile * kAKeys;
        uint64_t *bar = &full[warp][stage];
        vb_mbar_arrive_expect_tx(bar, Cfg::kStage);
        vb_bulk_g2s(to, a.c.k + row * (NB * 16), Cfg::kCodes, bar);
        vb_bulk_g2s(to + Cfg::kCodes, a.c.ks + row * NB, Cfg::kScales, bar);
        vb_bulk_g2s(to + Cfg::kCodes + Cfg::kScales, a.c.v + row * (NB * 16), Cfg::kCodes, bar);
        vb_bulk_g2s(to + 2 * Cfg::kCodes + Cfg::kScales, a.c.vs + row * NB, Cfg::kScales, bar);
    };
    if (lane == 0) {
        for (int i = 0; i < Cfg::kStages; i++) vb_mbar_init(&full[warp][i], 1);
        vb_mbar_init_fence();
        for (int i = 0; i < Cfg::kStages; i++)
            if (t_begin + i * kAWarps < t_end) fetch(t_begin + i * kAWarps, i);
    }
    if (tid == 0) abort_flag = 0;
    column.template put<QT>(a, warp, q_s, mul_s);
    __syncthreads();

    /* columns 2 t and 2 t + 1 of this lane: tokens they see, what makes their scores powers of two */
    int sees[2];
    float mul[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const int col = 2 * t + u;
        sees[u] = before + (pair0 + min(col, n_pairs - 1)) / a.group + 1;      /* columns beyond the last pair are zeros and go nowhere */
        mul[u] = mul_s[col];
    }
    const int all_see = before + pair0 / a.group + 1;                /* tokens that every column sees */

    float ref[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
    float o[2 * NB][4];
#pragma unroll
    for (int i = 0; i < 2 * NB; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) o[i][j] = 0.0f;
    int top_scale[kVS], first_scale[kVS];
    bool far = false;
#pragma unroll
    for (int i = 0; i < kVS; i++) top_scale[i] = first_scale[i] = 0;

    int stage = 0;
    uint32_t parity = 0;
    for (int tile = t_begin; tile < t_end; tile += kAWarps) {
        if (!__all_sync(0xffffffffu, vb_mbar_wait(&full[warp][stage], parity, &abort_flag))) {
            atomicCAS(a.status, 0, kAStatus);
            *(volatile int *)&abort_flag = 1;
            /* what is on its way lands before the memory is used for something else */
            volatile int stay = 0;
            for (int i = 0; i < Cfg::kStages && tile + i * kAWarps < t_end; i++) {
                vb_mbar_wait(&full[warp][stage], parity, &stay);
                if (++stage == Cfg::kStages) { stage = 0; parity ^= 1u; }
            }
            break;
        }
        const unsigned char *ks = ring + stage * Cfg::kStage, *kss = ks + Cfg::kCodes, *vs = kss + Cfg::kScales, *vss = vs + Cfg::kCodes;
        const int j0 = tile * kAKeys;

        /* scores */
        float s[2][4];
        {
            uint32_t w[2][2][NB];
            float f[2][2][NB];
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int key = m * 16 + u * 8 + g;
                    get_words<NB>(ks + key * (NB * 16) + t * (NB * 4), w[m][u]);
                    get_scales<NB>(kss + key * NB, f[m][u]);
                }
#pragma unroll
            for (int b = 0; b < NB; b++) {
                uint2 qf[2][QT];
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int u = 0; u < QT; u++) qf[h][u] = q_s[((b * 2 + h) * QT + u) * 32 + lane];
#pragma unroll
                for (int m = 0; m < 2; m++)
                    if (b == 0) block_scores<true, QT>(s[m], w[m][0][b], w[m][1][b], f[m][0][b], f[m][1][b], qf);
                    else block_scores<false, QT>(s[m], w[m][0][b], w[m][1][b], f[m][0][b], f[m][1][b], qf);
            }
        }
        const bool masked = j0 + kAKeys > all_see;
        if (masked) {
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (j0 + m * 16 + (j >> 1) * 8 + g >= sees[j & 1]) s[m][j] = -INFINITY;
        }
        float top[2];
#pragma unroll
        for (int u = 0; u < 2; u++) top[u] = fmaxf(fmaxf(s[0][u], s[0][2 + u]), fmaxf(s[1][u], s[1][2 + u])) * mul[u];      /* the factors are positive */
        if (__any_sync(0xffffffffu, top[0] > ref[0] + kKv4Trail || top[1] > ref[1] + kKv4Trail)) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) top[u] = fmaxf(top[u], __shfl_xor_sync(0xffffffffu, top[u], x));
                if (top[u] > ref[u] + kKv4Trail) {
                    const float fall = exp2_fast(ref[u] - top[u]);      /* the first time: 0 */
                    ref[u] = top[u];
                    sum[u] *= fall;
#pragma unroll
                    for (int i = 0; i < 2 * NB; i++) {
                        o[i][u] *= fall;
                        o[i][2 + u] *= fall;
                    }
                }
            }
            __syncwarp();                                /* columns rise by themselves; a transposition takes the whole warp */
        }
        /* weights, turned into the B operand of V^T P^T */
        uint2 p[2][PT];
        const float low0 = ref[0] > -INFINITY ? ref[0] - kKv4Bias : 0.0f, low1 = ref[1] > -INFINITY ? ref[1] - kKv4Bias : 0.0f;
#pragma unroll
        for (int m = 0; m < 2; m++) {
            float e[4];
#pragma unroll
            for (int j = 0; j < 4; j++) e[j] = exp2_fast(fmaf(s[m][j], mul[j & 1], (j & 1) ? -low1 : -low0));
            sum[0] += e[0] + e[2];
            sum[1] += e[1] + e[3];
            const uint32_t h0 = half_pack(e[0], e[1]), h1 = half_pack(e[2], e[3]);
            p[m][0] = make_uint2(mat_turn(h0), mat_turn(h1));
            if constexpr (PT == 2) {
                const float2 f0 = kv4_f2(h0), f1 = kv4_f2(h1);
                p[m][1] = make_uint2(mat_turn(half_pack(e[0] - f0.x, e[1] - f0.y)), mat_turn(half_pack(e[2] - f1.x, e[3] - f1.y)));
            }
        }

        /* values: tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of each 16; their scale bytes in pairs, the largest and the smallest of them */
        uint32_t vsc[2][2][kVS];
        int most[kVS], least[kVS];
#pragma unroll
        for (int i = 0; i < kVS; i++) {
            uint32_t hi = 0u, lo = 0x00ff00ffu;
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const unsigned char *at = vss + (m * 16 + x * 8 + 2 * t) * NB + (Cfg::kWhole ? g * NB / 8 : i);
                    vsc[m][x][i] = at[0] + 65536u * at[NB];
                }
            if (masked) {                                /* whatever lies behind the last token */
#pragma unroll
                for (int m = 0; m < 2; m++)
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        const int key = j0 + m * 16 + x * 8 + 2 * t;
                        vsc[m][x][i] = key + 1 < seen ? vsc[m][x][i] : key < seen ? vsc[m][x][i] & 0xffffu : 0u;
                    }
            }
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    hi = __vmaxu2(hi, vsc[m][x][i]);
                    lo = __vminu2(lo, vsc[m][x][i]);
                }
            most[i] = (int)max(hi & 0xffffu, hi >> 16);
            least[i] = (int)min(lo & 0xffffu, lo >> 16);
        }
        bool rise = false;
#pragma unroll
        for (int i = 0; i < kVS; i++) rise |= most[i] > top_scale[i];
        if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
            for (int i = 0; i < kVS; i++) {
                most[i] = max(most[i], __shfl_xor_sync(0xffffffffu, most[i], 1));
                most[i] = max(most[i], __shfl_xor_sync(0xffffffffu, most[i], 2));
                if (__any_sync(0xffffffffu, most[i] == 255)) {
                    /* a block that is NaN: so are the columns that see it; its codes are zeros */
                    int bad = 1 << 30;
                    most[i] = 0;
#pragma unroll
                    for (int m = 0; m < 2; m++)
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            const uint32_t at = 16u * (x & 1), byte = (vsc[m][x >> 1][i] >> at) & 0xffffu;
                            if (byte == 255u) {
                                bad = min(bad, j0 + m * 16 + (x >> 1) * 8 + 2 * t + (x & 1));
                                vsc[m][x >> 1][i] &= ~(0xffffu << at);
                                least[i] = 0;
                            } else {
                                most[i] = max(most[i], (int)byte);
                            }
                        }
#pragma unroll
                    for (int x = 1; x < 4; x <<= 1) {
                        bad = min(bad, __shfl_xor_sync(0xffffffffu, bad, x));
                        most[i] = max(most[i], __shfl_xor_sync(0xffffffffu, most[i], x));
                    }
#pragma unroll
                    for (int r = 0; r < 2 * NB; r++)
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            if ((Cfg::kWhole || r / 2 == i) && bad < sees[j & 1]) o[r][j] = __uint_as_float(0x7fffffffu);
                }
                const int up = most[i] - top_scale[i];
                if (up > 0) {
                    const float fall = up > 126 ? 0.0f : __uint_as_float((uint32_t)(127 - up) << 23);
                    if (top_scale[i] == 0) first_scale[i] = most[i];
                    top_scale[i] = most[i];
                    far |= most[i] - first_scale[i] > kKv4Rise;
#pragma unroll
                    for (int r = 0; r < 2 * NB; r++)
                        if (Cfg::kWhole || r / 2 == i) {
#pragma unroll
                            for (int j = 0; j < 4; j++) o[r][j] *= fall;
                        }
                }
            }
        }
        /* 2^(byte - top + 13) in FP16: an exponent field of byte - top + 28, two at a time, where that is a normal number for all */
        bool deep = false;
#pragma unroll
        for (int i = 0; i < kVS; i++) deep |= least[i] + 27 < top_scale[i];
        if (!__any_sync(0xffffffffu, deep)) {
#pragma unroll
            for (int i = 0; i < kVS; i++) {
                const uint32_t add = (uint32_t)(28 - top_scale[i]) * 0x04000400u;
#pragma unroll
                for (int m = 0; m < 2; m++)
#pragma unroll
                    for (int x = 0; x < 2; x++) vsc[m][x][i] = vsc[m][x][i] * 1024u + add;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kVS; i++)
#pragma unroll
                for (int m = 0; m < 2; m++)
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        far |= kv4_far(vsc[m][x][i] & 0xffffu, top_scale[i]) || kv4_far(vsc[m][x][i] >> 16, top_scale[i]);
                        const int lo = (int)(vsc[m][x][i] & 0xffffu) + 140 - top_scale[i], hi = (int)(vsc[m][x][i] >> 16) + 140 - top_scale[i];
                        vsc[m][x][i] = half_pack(__uint_as_float((uint32_t)max(lo, 0) << 23), __uint_as_float((uint32_t)max(hi, 0) << 23));
                    }
        }
#pragma unroll
        for (int m = 0; m < 2; m++) {
            const uint32_t (&f)[2][kVS] = vsc[m];
            uint32_t w[4][kW];
#pragma unroll
            for (int x = 0; x < 4; x++) get_values<NB>(vs + (m * 16 + (x >> 1) * 8 + 2 * t + (x & 1)) * (NB * 16) + g * (NB * 2), w[x]);
#pragma unroll
            for (int i = 0; i < kW; i++) {
                uint32_t r[2][2][4];                    /* [token pair][value of the byte][byte]: the two tokens' values side by side */
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const uint32_t wa = w[2 * x][i], wb = w[2 * x + 1][i];
                    kv4_halves((wa & 0x0f0f0f0fu) | ((wb << 4) & 0xf0f0f0f0u), r[x][0]);
                    kv4_halves(((wa >> 4) & 0x0f0f0f0fu) | (wb & 0xf0f0f0f0u), r[x][1]);
                }
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int at = i * 4 + k, sc = Cfg::kWhole ? 0 : at / 2;
                    if (at < 2 * NB) {
                        const uint32_t a0 = half_mul(r[0][0][k], f[0][sc]), a1 = half_mul(r[0][1][k], f[0][sc]);
                        const uint32_t a2 = half_mul(r[1][0][k], f[1][sc]), a3 = half_mul(r[1][1][k], f[1][sc]);
                        if constexpr (kExact) {
                            float c[4];
                            mma_f16_first(c, a0, a1, a2, a3, p[m][0]);
#pragma unroll
                            for (int u = 1; u < PT; u++) mma_f16(c, a0, a1, a2, a3, p[m][u]);
                            const float2 lo = vb_f2_get(vb_f2_add(vb_f2_pack(o[at][0], o[at][1]), vb_f2_pack(c[0], c[1])));
                            const float2 hi = vb_f2_get(vb_f2_add(vb_f2_pack(o[at][2], o[at][3]), vb_f2_pack(c[2], c[3])));
                            o[at][0] = lo.x; o[at][1] = lo.y; o[at][2] = hi.x; o[at][3] = hi.y;
                        } else {
#pragma unroll
                            for (int u = 0; u < PT; u++) mma_f16(o[at], a0, a1, a2, a3, p[m][u]);
                        }
                    }
                }
            }
        }
        __syncwarp();
        if (lane == 0 && tile + Cfg::kStages * kAWarps < t_end) fetch(tile + Cfg::kStages * kAWarps, stage);
        if (++stage == Cfg::kStages) { stage = 0; parity ^= 1u; }
    }

    /* the warps' parts together, in the order of the accumulators (conflict-free, and the same place is the same result for all);
     * sums and results lose the 2^15 that the weights may have */
#pragma unroll
    for (int u = 0; u < 2; u++) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], x);
        sum[u] *= kKv4Out;
    }
    const bool plain = __syncthreads_or(far);            /* every ring is empty */
    constexpr int kUnits = 2 * NB * 32;                  /* of four results */
    float4 *mo = reinterpret_cast<float4 *>(a_smem);
    float2 *mm = reinterpret_cast<float2 *>(mo + kAWarps * kUnits), *ml = mm + kAWarps * 4;
    if (g == 0) {
        mm[warp * 4 + t] = make_float2(ref[0], ref[1]);
        ml[warp * 4 + t] = make_float2(sum[0], sum[1]);
    }
#pragma unroll
    for (int i = 0; i < 2 * NB; i++) {
        const int e = top_scale[Cfg::kWhole ? 0 : i / 2] - kKv4Down, e0 = e >> 1;      /* in two steps: 2^e may not be a normal number */
        const float f0 = __uint_as_float((uint32_t)(127 + e0) << 23), f1 = __uint_as_float((uint32_t)(127 + e - e0) << 23);
        mo[(warp * 2 * NB + i) * 32 + lane] = make_float4(o[i][0] * f0 * f1, o[i][1] * f0 * f1, o[i][2] * f0 * f1, o[i][3] * f0 * f1);
    }
    __syncthreads();
    constexpr int kPart = kACols * (kDim + 2);           /* floats of a part: results, references, sums */
    const int stride = (pairs + kACols - 1) / kACols * a.c.kv_heads, first_cta = (int)blockIdx.x - split * stride;       /* of this unit; its parts lie so many CTAs apart */
    float *parts = a.part + (size_t)first_cta * kPart;
    const size_t step = (size_t)stride * kPart;
    /* four results of columns 2 t, 2 t + 1 and dims d, d + 1, against a reference and a sum each */
    auto finish = [&](int i, float4 v, float2 total, float2 reference) {
        const int d = Cfg::kWhole ? g * (4 * NB) + 2 * i : 32 * (i / 2) + 4 * g + 2 * (i & 1);
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int col = 2 * t + u, pair = pair0 + col;
            if (col >= n_pairs) continue;
            const float l = u ? total.y : total.x, r = u ? reference.y : reference.x, inv = l == 0.0f ? 0.0f : 1.0f / l;
            const float x = l == 0.0f ? 0.0f : (u ? v.y : v.x) * inv, y = l == 0.0f ? 0.0f : (u ? v.w : v.z) * inv;
            const int row = pair / a.group, head = kv_head * a.group + pair - row * a.group;
            T *to = out.data + seq * out.seq + row * out.row + head * out.head + d;
            if (a.wide_out) {
                if constexpr (sizeof(T) == 4) *reinterpret_cast<float2 *>(to) = make_float2(x, y);
                else *reinterpret_cast<uint32_t *>(to) = serve_pack(x, y, to);
            } else {
                serve_put(to, x);
                serve_put(to + 1, y);
            }
            if (d == 0 && a.lse) a.lse[((size_t)seq * a.max_rows + row) * a.heads + head] = l == 0.0f ? -INFINITY : (r + (float)kKv4Rest + log2f(l)) * 0.69314718f;
        }
    };
    /* a part's factor against a reference; parts without weights have none */
    auto factor = [](float m, float reference) { return m > -INFINITY || m != m ? exp2_fast(m - reference) : 0.0f; };
    if (plain) {
        __syncthreads();
        const int pair = pair0 + warp, row = pair / a.group, head = kv_head * a.group + pair - row * a.group;
        const int tok0 = used == 1 ? 0 : split * share * kAKeys;
        if (warp < n_pairs) {
            float *q_row = reinterpret_cast<float *>(a_smem) + warp * 2 * kDim, *results = q_row + kDim;
            const float2 end = kv4_plain_row<NB, T>(kv4_head<NB>(a.c, row0), q.data + seq * q.seq + row * q.row + head * q.head, a.scale, tok0,
                                                    min(min(t_end * kAKeys, seen), before + row + 1), q_row, results);
            float *part = parts + split * step;
            const float inv = end.y == 0.0f ? 0.0f : 1.0f / end.y;
            for (int d = lane; d < kDim; d += 32) {
                if (used == 1) {
                    serve_put(out.data + seq * out.seq + row * out.row + head * out.head + d, end.y == 0.0f ? 0.0f : results[d] * inv);
                } else {                                 /* in the accumulators' order */
                    const int gd = Cfg::kWhole ? d / (4 * NB) : d % 32 / 4, i = Cfg::kWhole ? d % (4 * NB) / 2 : d / 32 * 2 + d % 4 / 2;
                    part[((i * 32 + gd * 4 + (warp >> 1)) * 2 + (d & 1)) * 2 + (warp & 1)] = results[d];
                }
            }
            if (lane == 0 && used == 1 && a.lse) a.lse[((size_t)seq * a.max_rows + row) * a.heads + head] = end.y == 0.0f ? -INFINITY : (end.x + (float)kKv4Rest + log2f(end.y)) * 0.69314718f;
            if (lane == 0 && used > 1) {
                part[kACols * kDim + warp] = end.x;
                part[kACols * kDim + 8 + warp] = end.y;
            }
        }
        if (used == 1) return;
    } else {
        float2 reference = make_float2(-INFINITY, -INFINITY), total = make_float2(0.0f, 0.0f), f[kAWarps];
#pragma unroll
        for (int w = 0; w < kAWarps; w++) {
            f[w] = mm[w * 4 + t];
            reference.x = fmaxf(reference.x, f[w].x);
            reference.y = fmaxf(reference.y, f[w].y);
        }
#pragma unroll
        for (int w = 0; w < kAWarps; w++) {
            const float2 l = ml[w * 4 + t];
            f[w] = make_float2(factor(f[w].x, reference.x), factor(f[w].y, reference.y));
            total.x += l.x * f[w].x;
            total.y += l.y * f[w].y;
        }
        for (int i = warp; i < 2 * NB; i += kAWarps) {
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kAWarps; w++) {
                const float4 x = mo[(w * 2 * NB + i) * 32 + lane];
                v.x = fmaf(x.x, f[w].x, v.x);
                v.y = fmaf(x.y, f[w].y, v.y);
                v.z = fmaf(x.z, f[w].x, v.z);
                v.w = fmaf(x.w, f[w].y, v.w);
            }
            if (used == 1) finish(i, v, total, reference);
            else reinterpret_cast<float4 *>(parts + split * step)[i * 32 + lane] = v;
        }
        if (used == 1) return;
        if (warp == 0 && g == 0) {
            float2 *to = reinterpret_cast<float2 *>(parts + split * step + kACols * kDim);
            to[t] = reference;
            to[4 + t] = total;
        }
    }
    /* the CTA that comes last joins the parts, in their order whoever that is */
    __threadfence();
    __syncthreads();
    if (tid == 0) {
        is_last = atomicAdd(&a.tickets[first_cta], 1u) == (unsigned)used - 1u;
        if (is_last) a.tickets[first_cta] = 0u;
        __threadfence();
    }
    __syncthreads();
    if (!is_last) return;
    float2 *ends = reinterpret_cast<float2 *>(a_smem);               /* references and sums of all parts; then factors in their place */
    for (int x = tid; x < used * 8; x += kAThreads) ends[x] = __ldcg(reinterpret_cast<const float2 *>(parts + (x >> 3) * step + kACols * kDim) + (x & 7));
    __syncthreads();
    float2 reference = make_float2(-INFINITY, -INFINITY), total = make_float2(0.0f, 0.0f);
    for (int w = 0; w < used; w++) {
        const float2 m = ends[w * 8 + t];
        reference.x = fmaxf(reference.x, m.x);
        reference.y = fmaxf(reference.y, m.y);
    }
    for (int w = 0; w < used; w++) {
        const float2 m = ends[w * 8 + t], l = ends[w * 8 + 4 + t];
        total.x += l.x * factor(m.x, reference.x);
        total.y += l.y * factor(m.y, reference.y);
    }
    for (int i = warp; i < 2 * NB; i += kAWarps) {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int w = 0; w < used; w++) {
            const float4 x = __ldcg(reinterpret_cast<const float4 *>(parts + w * step) + i * 32 + lane);
            const float2 m = ends[w * 8 + t];
            const float fx = factor(m.x, reference.x), fy = factor(m.y, reference.y);
            v.x = fmaf(x.x, fx, v.x);
            v.y = fmaf(x.y, fy, v.y);
            v.z = fmaf(x.z, fx, v.z);
            v.w = fmaf(x.w, fy, v.w);
        }
        finish(i, v, total, reference);
    }
}

/* mass_out: the scores again, now that the rows' sums are known (in the attention kernel only the last CTA of a split sequence knows them,
 * and keeping scores takes memory for every row). A CTA has up to four tiles of tokens a warp, whose keys stay in shared memory while the
 * (row, head) pairs come by, 64 at a time, a column of eight by each warp. A token's weights are summed in one order: no atomics. One row of 32
 * heads over eight sequences of 4608 tokens and 8 KV heads of 128, bf16: 17 us by itself where the attention takes 20, 32 both, whose ends overlap. */
constexpr int kMTiles = 4, kMMostPairs = 64;      /* of a KV head: more take the kernel of vb_kv4_prompt.cu, heads up to 128 */

template <int NB, class T>
struct MCfg {
    static constexpr int QT = sizeof(T) == 4 ? 2 : 1;
    static constexpr int kTile = kAKeys * NB * 17;                                  /* codes, scales */
    static constexpr int kQ = NB * 2 * QT * 32 * 8;                                 /* eight pairs */
    static constexpr int smem(int tiles) { return kAWarps * (tiles * kTile + kQ); }
};

template <int NB, class T>
__global__ void __launch_bounds__(kAThreads, NB <= 4 ? 2 : 1) kv4_mass_kernel(const Kv4Attn a, const ServeRows<T> q, int warp_tiles) {
    using Cfg = MCfg<NB, T>;
    constexpr int QT = Cfg::QT;
    extern __shared__ __align__(128) unsigned char a_smem[];
    __shared__ __align__(8) uint64_t full[kAWarps];
    __shared__ float mul_s[kAWarps * kACols], lse_s[kAWarps * kACols];
    __shared__ int abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int kv_head = blockIdx.y, seq = blockIdx.z;
    /* begins beside the end of the attention kernel, which has waited for all that is read here but the rows' sums; masses may not
     * be written before those are waited for either */
    const bool alone = a.max_rows == 0;
    if (alone) pdl_wait();
    const Kv4Span span = kv4_span(a.lengths, a.rows, a.max_rows, seq, a.c.capacity);
    const int pairs = span.rows * a.group, before = span.length - span.rows;
    const int cta0 = blockIdx.x * kAWarps * warp_tiles * kAKeys;
    if (cta0 >= span.length) {
        if (!alone) pdl_wait();    /* no launch is over before the ones it follows are */
        return;
    }
    const int tile0 = (blockIdx.x * kAWarps + warp) * warp_tiles, tiles = min(warp_tiles, (span.length + kAKeys - 1) / kAKeys - tile0);
    unsigned char *keys = a_smem + warp * warp_tiles * Cfg::kTile;
    uint2 *q_s = reinterpret_cast<uint2 *>(a_smem + kAWarps * warp_tiles * Cfg::kTile);
    if (lane == 0) {
        vb_mbar_init(&full[warp], 1);
        vb_mbar_init_fence();
        if (tiles > 0) {
            const size_t row = a.c.row(seq, kv_head, tile0 * kAKeys);
            vb_mbar_arrive_expect_tx(&full[warp], tiles * Cfg::kTile);
            vb_bulk_g2s(keys, a.c.k + row * (NB * 16), tiles * kAKeys * NB * 16, &full[warp]);
            vb_bulk_g2s(keys + warp_tiles * kAKeys * NB * 16, a.c.ks + row * NB, tiles * kAKeys * NB, &full[warp]);
        }
    }
    if (tid == 0) abort_flag = 0;
    __syncthreads();
    float mass[kMTiles][2][2];
#pragma unroll
    for (int i = 0; i < kMTiles; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) mass[i][j >> 1][j & 1] = 0.0f;
    bool here = tiles <= 0, waited = alone;
    /* rows before this CTA's first token see none of its tokens */
    for (int group0 = max(0, cta0 - before) * a.group / kACols * kACols; group0 < pairs; group0 += kAWarps * kACols) {
        __syncthreads();                                                            /* the pairs before are done with */
        const int made = min(kAWarps, (pairs - group0 + kACols - 1) / kACols);
#pragma unroll 1
        for (int r = 0; r < made; r++) {
            QueryColumn<NB, T> column;
            column.load(q, a, seq, kv_head, group0 + r * kACols + warp, pairs);
            column.template put<QT>(a, warp, q_s + r * (Cfg::kQ / 8), mul_s + r * kACols);
        }
        if (!waited) pdl_wait();
        waited = true;
        if (tid < kAWarps * kACols) {
            const int pair = group0 + tid, row = pair / a.group;
            const float lse = pair < pairs ? a.lse[((size_t)seq * a.max_rows + row) * a.heads + kv_head * a.group + pair - row * a.group] : 0.0f;
            lse_s[tid] = lse == -INFINITY ? INFINITY : lse * 1.44269504f;           /* a row without weights gives none */
        }
        __syncthreads();
        if (!here) {
            if (!__all_sync(0xffffffffu, vb_mbar_wait(&full[warp], 0u, &abort_flag))) {
                atomicCAS(a.status, 0, kAStatus);
                *(volatile int *)&abort_flag = 1;
                volatile int stay = 0;
                vb_mbar_wait(&full[warp], 0u, &stay);
            }
            here = true;
        }
#pragma unroll
        for (int i = 0; i < kMTiles; i++) {
            if (i >= tiles) break;
            const unsigned char *ks = keys + i * kAKeys * NB * 16, *kss = keys + (warp_tiles * 16 + i) * kAKeys * NB;
            const int j0 = (tile0 + i) * kAKeys;
            uint32_t w[2][2][NB];
            float f[2][2][NB];
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int key = m * 16 + u * 8 + g;
                    get_words<NB>(ks + key * (NB * 16) + t * (NB * 4), w[m][u]);
                    get_scales<NB>(kss + key * NB, f[m][u]);
                }
#pragma unroll 1
            for (int r = 0; r < made; r++) {
                float s[2][4];
                __syncwarp();                            /* lanes differ in what they have added up */
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    uint2 qf[2][QT];
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int u = 0; u < QT; u++) qf[h][u] = q_s[r * (Cfg::kQ / 8) + ((b * 2 + h) * QT + u) * 32 + lane];
#pragma unroll
                    for (int m = 0; m < 2; m++)
                        if (b == 0) block_scores<true, QT>(s[m], w[m][0][b], w[m][1][b], f[m][0][b], f[m][1][b], qf);
                        else block_scores<false, QT>(s[m], w[m][0][b], w[m][1][b], f[m][0][b], f[m][1][b], qf);
                }
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int col = r * kACols + 2 * t + u, pair = group0 + col;
                    const int sees = pair < pairs ? before + pair / a.group + 1 : 0;
                    const float mul = mul_s[col], lse = lse_s[col];
#pragma unroll
                    for (int m = 0; m < 2; m++)
#pragma unroll
                        for (int k = 0; k < 2; k++)
                            if (j0 + m * 16 + k * 8 + g < sees) mass[i][m][k] += exp2_fast(s[m][2 * k + u] * mul - lse);
                }
            }
        }
    }
    if (!waited) pdl_wait();
    if (!here) vb_mbar_wait(&full[warp], 0u, &abort_flag);                          /* no rows: nothing leaves while its keys are on their way */
    const size_t base = ((size_t)seq * a.c.kv_heads + kv_head) * a.c.capacity;
#pragma unroll
    for (int i = 0; i < kMTiles; i++) {
        if (i >= tiles) break;
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
                float v = mass[i][m][r];
                v += __shfl_xor_sync(0xffffffffu, v, 1);
                v += __shfl_xor_sync(0xffffffffu, v, 2);
                const int j = (tile0 + i) * kAKeys + m * 16 + r * 8 + g;
                if (t == 0 && j < span.length) a.mass_out[base + j] = v + (a.mass_in && j < before ? a.mass_in[base + j] : 0.0f);
            }
    }
}

template <int NB, class T>
int attn_launch(const Kv4Attn &args, const vb200_kv4_attention_t &v, const Kv4Work &work, cudaStream_t st) {
    using Cfg = ACfg<NB>;
    constexpr int PT = kWeightTerms<T>;
    Kv4Attn a = args;
    const ServeRows<T> q = serve_rows<T>(v.q), out = serve_rows<T>(v.out);
    a.wide = serve_wide(q);
    a.wide_out = serve_wide(out);
    /* Eight pairs against n tokens cost 32 ps n here and 128 pairs 181 ps n on the tensor cores' kernel, which takes 17 us more to begin
     * and to join (fp32, heads of 128; the other types and sizes cross at about the same place). Measured, here and there in us: 8 heads, 1024
     * tokens, 256 and 512 pairs each 17, 30 and 29, 39; 8192 tokens, 64 and 128 pairs 31, 52 and 33, 44; 65536 tokens, 32 and 64 pairs 86, 176 and
     * 107, 110; 64 heads, 1024 tokens, 64 and 128 pairs 31, 52 and 35, 46. The tokens are the cache's room for them: lengths are not
     * known here, and those figures are of full caches. Where most of the room is empty the other kernel is taken from fewer tokens on than it
     * pays for: its 17 us. */
    const long long pairs = (long long)a.max_rows * a.group, room = (long long)a.c.capacity * a.c.kv_heads * a.c.seqs;
    if (NB <= 4 && (double)room * (double)((pairs + 7) / 8 - 6 * ((pairs + 127) / 128)) > 550e3) {
        if (kv4_prompt(a, q, out, work.sm_count, st)) return -1;
    } else if (a.max_rows > 0) {
        const long long row_tiles = ((long long)a.max_rows * a.group + kACols - 1) / kACols;
        const long long units = row_tiles * a.c.kv_heads * a.c.seqs, at_once = (long long)work.sm_count * (NB <= 4 ? 2 : 1);
        if (units > INT_MAX) return serve_fail("too many rows");
        a.row_tiles = (int)row_tiles;
        a.split = units < at_once && a.c.capacity > 2 * kAWarps * kAKeys;
        if (launch_pdl(kv4_attn_kernel<NB, PT, T>, dim3((unsigned)(a.split ? at_once : units)), dim3(kAThreads), Cfg::kBig, st, a, q, out) != cudaSuccess)
            return serve_launched() | -1;
    }
    if (a.mass_out && NB <= 4 && pairs > kMMostPairs) return kv4_mass_many(a, q, st);
    if (a.mass_out) {
        /* the more tiles a warp has, the fewer CTAs make the queries: as many as leave every SM one */
        const long long heads = (long long)a.c.kv_heads * a.c.seqs, tiles = ((long long)a.c.capacity + kAKeys - 1) / kAKeys;
        int warp_tiles = kMTiles;
        while (warp_tiles > 1 && (tiles + kAWarps * warp_tiles - 1) / (kAWarps * warp_tiles) * heads < work.sm_count) warp_tiles >>= 1;
        const dim3 grid((unsigned)((tiles + kAWarps * warp_tiles - 1) / (kAWarps * warp_tiles)), a.c.kv_heads, a.c.seqs);
        if (launch_pdl(kv4_mass_kernel<NB, T>, grid, dim3(kAThreads), MCfg<NB, T>::smem(warp_tiles), st, a, q, warp_tiles) != cudaSuccess)
            return serve_launched() | -1;
    }
    return 0;
}

template <class T>
int attn_dims(const Kv4Attn &a, const vb200_kv4_attention_t &v, const Kv4Work &w, cudaStream_t st) {
#define VB_CALL(n) attn_launch<n, T>(a, v, w, st)
    VB_KV4_DIMS(a.c.blocks, VB_CALL)
#undef VB_CALL
}

/* Loads the kernels of a head size on the current device, and lets them have their shared memory. */
template <int NB, class T>
int attn_load() {
    return cudaFuncSetAttribute(kv4_attn_kernel<NB, kWeightTerms<T>, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, ACfg<NB>::kBig) == cudaSuccess &&
                   cudaFuncSetAttribute(kv4_mass_kernel<NB, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, MCfg<NB, T>::smem(kMTiles)) == cudaSuccess
               ? 0
               : -1;
}

} // namespace

int kv4_attention_load(int blocks) {
    if (kv4_prompt_load(blocks)) return -1;
#define VB_CALL(n) (attn_load<n, float>() || attn_load<n, __nv_bfloat16>() || attn_load<n, __half>() ? serve_launched() | -1 : 0)
    VB_KV4_DIMS(blocks, VB_CALL)
#undef VB_CALL
}

int kv4_attention(const Kv4 &c, const Kv4Work &w, const vb200_kv4_attention_t &v, cudaStream_t st) {
    Kv4Attn a = {};
    a.c = c;
    a.lengths = v.lengths; a.rows = v.rows; a.max_rows = v.max_rows; a.heads = v.heads; a.group = v.heads / c.kv_heads;
    a.scale = v.scale; a.lse = v.lse; a.mass_in = v.mass_in; a.mass_out = v.mass_out;
    a.part = w.part; a.aside = w.aside; a.tickets = w.tickets; a.rooms = w.rooms; a.n_rooms = w.sm_count; a.status = w.status;
    if ((long long)a.max_rows * a.group > (1ll << 30)) return serve_fail("too many rows");
    if (v.q.type == VB200_F32) return attn_dims<float>(a, v, w, st);
    if (v.q.type == VB200_BF16) return attn_dims<__nv_bfloat16>(a, v, w, st);
    return attn_dims<__half>(a, v, w, st);
}

} // namespace vb

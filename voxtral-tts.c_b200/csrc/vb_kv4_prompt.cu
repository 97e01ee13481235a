/*
 * vb_kv4_prompt.cu - softmax attention over the 4-bit cache for many rows, on the 5th-generation tensor cores.
 *
 * A CTA owns one KV head and 128 (row, query head) pairs and walks the tokens 128 at a time:
 *
 *   S [128 x 128]   = Q K^T    Q in shared memory, one FP16 term (bf16, fp16) or two (fp32), rows brought to [2^14, 2^15)
 *   O [128 x dim]  += P V      P in TMEM, in S's own columns, one term (bf16) or two; V rows [token][dim] are an MN-major operand
 *
 * Keys and values go from codes to FP16 on the way to shared memory, four warps for the keys and three for the values: keys times
 * 2^(e - S + 13), S the largest scale of a warp's 32 tokens, which the softmax undoes, values times 2^(e - E + 13), E the largest scale
 * so far, on which the accumulator is based: exact down to 2^-36 of the largest. A CTA that meets others works in fp32 (p_plain). Scores,
 * weights, sums as in vb_kv4_attn.cu. Two pairs of
 * warpgroups take alternate tiles with a reference, sums and an accumulator each, merged at the end, so that the tensor pipe works on
 * one tile while the other is in its softmax. A thread has half of a row's columns: with a whole row a thread, and half as many
 * threads, 1203 rows took 206 us in place of 178 (before sums were put aside).
 * Nothing is saturated: a tile of 128 x 128 takes an SM 5800 clocks with two terms each, of which the tensor pipe needs 2048 (36 %; 26 % for bf16); issue
 * slots are 50 % busy, the integer pipe 41. The roles wait for one another: scores for keys, the softmax for scores and for the other half of its
 * rows, results for all of a tile's weights. 1203 fp32 rows of 32 heads of 128 over 4208 tokens: 204 us, 349 TFLOP/s (twice that as executed);
 * 1024 bf16 rows over 4096 tokens 123 us.
 *
 * Warps: 0-7, 8-15 softmax, 16-19 keys, 20-22 values, 23 issues the MMAs. All waits are bounded.
 */
#include <algorithm>

#include "vb_attn_tc.cuh"
#include "vb_kv4.cuh"

namespace vb {

namespace {

constexpr int kPRows = 128, kPKeys = 128, kPSoft = 512, kPMmaWarp = 23, kPThreads = 32 * (kPMmaWarp + 1), kPBlock = kPKeys * 128, kPStatus = 62, kPRing = 8;
constexpr int kPLeast = 2, kPTailParts = 8;   /* tiles of a part at least; parts of a unit of the last round at most */
constexpr uint32_t kPTmem = 512, kPO = 256;
/* A row's reference trails by at most 2^4 here, weights are held times 2^11. With 2^2 and 2^13, as in vb_kv4_attn.cu, more tiles change a reference of
 * one of a warp's 32 rows: 1024 bf16 rows over 4096 tokens 133 us in place of 126, 1203 fp32 rows over 4208 213 in place of 207. */
constexpr float kPTrail = 4.0f, kPBias = 11.0f, kPOut = 0x1p-19f;
constexpr int kPDown = 127 + 13 + 19;
template <int NB, int QT>
struct PCfg {
    /* A sum in TMEM loses up to a unit of its last place with every product of 16 tokens that is added, towards zero: 224 of them, 14 tiles of two
     * terms, left results of a portion of 1203 fp32 rows 3.4e-6 off 64 bits (elementary fp32 operations: 1.2e-6). So a warpgroup pair puts what
     * a few tiles have made aside in global memory, added up there rounded to nearest. fp32: three tiles (six: 1.5e-6 off over 2112
     * tokens, where elementary operations are 0.7e-6 and three 0.9e-6). 1203 rows: 205 us, 195 with six, 177 without. Types that round
     * their results to less: 64. That leaves fp16 results over 32800 tokens 2.4e-5 lower than eight tiles do, a twentieth of half a unit (with
     * eight, 1024 rows over 4096 tokens take 157 us in place of 143); bf16 has half as many products, and a half unit eight times as large. */
    static constexpr int kChain = QT == 2 ? 3 : 64;
    static constexpr int kD64 = (NB + 1) / 2;                                  /* blocks of 64 columns */
    static constexpr int kSlot = kD64 * kPBlock;
    static constexpr int kSlots = kD64 >= 2 ? 2 : 3;
    static constexpr int kQ = QT * kSlot;
    static constexpr int kSmem = kQ + 2 * kSlots * kSlot + 1024;
    static constexpr int kPart = kPRows * (NB * 32 + 2);                       /* floats of a part: results, references and sums */
    static constexpr int kLd = NB * 32 + 4;                                    /* results on their way out: a row */
    static_assert(kPRows * kLd * 4 + 4 * kPRows * 16 <= 2 * kSlots * kSlot, "results do not fit the rings");
    static_assert(kSmem <= 232448 - 4096, "over what a CTA may use");
};

VB_DEVINL uint64_t p_desc_mn(uint32_t addr) {
    uint64_t d = (uint64_t)((addr >> 4) & 0x3FFF);
    d |= (uint64_t)(kPBlock >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
/* kind::f16 with FP16 operands, fp32 sums, 128 rows, n columns */
VB_DEVINL uint32_t p_idesc(int n, bool mn_major) { return (1u << 4) | (mn_major ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kPRows >> 4) << 24); }

/* 16 columns of this thread's TMEM lane */
template <int N>
VB_DEVINL void p_st16(uint32_t taddr, const uint32_t (&r)[N]) {
    static_assert(N >= 16, "");
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::VB_AT_R8(r, 0),
                 VB_AT_R8(r, 8), "r"(taddr)
                 : "memory");
}
/* Eight codes times a power of two to 16 bytes */
VB_DEVINL uint4 p_halves(uint32_t w, uint32_t f) {
    uint32_t r[4];
    kv4_halves(w, r);
    return make_uint4(half_mul(r[0], f), half_mul(r[1], f), half_mul(r[2], f), half_mul(r[3], f));
}
/* 2^(byte - top + 13) twice; byte <= top */
VB_DEVINL uint32_t p_factor(int byte, int top) {
    const float f = __uint_as_float((uint32_t)max(byte + 140 - top, 0) << 23);
    return half_pack(f, f);
}

/* What a CTA has: a unit's tiles of tokens, or the split-th part of them, and where its part lies and those beside it. */
struct PWork {
    int seq, kv_head, pair0, n_pairs, before, seen, used, split, first_tile, n_tiles, slot, stride;
    Kv4Span span;
};
/* Where there are fewer units than SMs, CTAs have shares of the work (kv4_place). Otherwise a CTA has a unit, but the units that would be
 * alone in a last round are cut into a.tail_parts (304 units of 24 to 33 tiles on 148 SMs: 206 us with three rounds). False: nothing. */
VB_DEVINL bool p_work(const Kv4Attn &a, int block, PWork &p) {
    int unit, share = INT_MAX, parts = 0;
    if (a.split) {
        const Kv4Place place = kv4_place<kPRows, kPKeys>(a, 1, kPLeast, kPRows);
        p.seq = place.seq; unit = place.unit; p.split = place.split; share = place.share; p.slot = block;
    } else {
        const int i = block - a.tail0, u = i < 0 ? block : a.tail0 + i % a.tail_units, units = a.row_tiles * a.c.kv_heads;
        p.seq = u / units;
        unit = u - p.seq * units;
        p.slot = i;
        p.split = i < 0 ? 0 : i / a.tail_units;
        parts = i < 0 ? 0 : a.tail_parts;
    }
    if (p.seq >= a.c.seqs) return false;
    p.span = kv4_span(a.lengths, a.rows, a.max_rows, p.seq, a.c.capacity);
    const int pairs = p.span.rows * a.group, row_tiles = (pairs + kPRows - 1) / kPRows, u = unit / a.c.kv_heads, tile_r = row_tiles - 1 - u;
    if (tile_r < 0) return false;                                  /* the latest rows see the most tokens: they go first */
    p.kv_head = unit - u * a.c.kv_heads;
    p.stride = a.split ? row_tiles * a.c.kv_heads : a.tail_units;
    p.pair0 = tile_r * kPRows;
    p.n_pairs = min(kPRows, pairs - p.pair0);
    p.before = p.span.length - p.span.rows;
    p.seen = max(0, p.before + (p.pair0 + p.n_pairs - 1) / a.group + 1);
    const int tiles = (p.seen + kPKeys - 1) / kPKeys;
    if (parts) share = max(kPLeast, (tiles + parts - 1) / parts);
    p.used = tiles <= share ? 1 : (tiles + share - 1) / share;
    p.first_tile = p.used == 1 ? 0 : p.split * share;
    p.n_tiles = p.used == 1 ? tiles : min(tiles, p.first_tile + share) - p.first_tile;
    return p.split < p.used;
}

/* Room for sums put aside, which a CTA takes for its time: as many as SMs, and a CTA has an SM to itself (its registers leave room for no
 * other), so that one is free. The SM's number is only where the search begins. False: none found, which would be a fault. */
VB_DEVINL bool p_take(const Kv4Attn &a, int &room) {
    uint32_t sm;
    asm("mov.u32 %0, %%smid;" : "=r"(sm));
    room = (int)(sm % (uint32_t)a.n_rooms);
    for (int i = 0; i < 1 << 16; i++) {
        if (atomicCAS(&a.rooms[room], 0u, 1u) == 0u) {
            __threadfence();
            return true;
        }
        room = room + 1 == a.n_rooms ? 0 : room + 1;
    }
    return false;
}
/* In it 32 columns of a warpgroup pair: [four columns][row], a float4 each. */
template <int NB>
VB_DEVINL float4 *p_aside(const Kv4Attn &a, int room, int pair, int block) {
    return reinterpret_cast<float4 *>(a.aside) + (((size_t)room * 2 + pair) * NB + block) * 8 * kPRows;
}

/* What is in TMEM is added to what lies aside, at the reference and scale of what is there unless those have come to lie too far below. A
 * function of its own: within the softmax its registers made that spill (1203 rows: 213 us in place of 207). */
template <int NB>
__device__ __noinline__ void p_put_aside(float4 *mine, float2 *base, uint32_t tO, int half, bool first, float ref, int top_scale) {
    const float2 there = *base;
    const int rises = top_scale - __float_as_int(there.y);
    const bool rebase = !first && (!(there.x > -INFINITY) || ref - there.x + (float)rises > 60.0f);
    const float g = first || rebase ? 1.0f : exp2_fast(ref - there.x) * __uint_as_float((uint32_t)(127 + rises) << 23);
    if (rebase) {
        const float fa = !(there.x > -INFINITY) || rises > 126 ? 0.0f : exp2_fast(there.x - ref) * __uint_as_float((uint32_t)(127 - rises) << 23);
#pragma unroll 1
        for (int c = half; c < NB; c += 2)
#pragma unroll 1
            for (int k = 0; k < 8; k++) {
                float4 *to = mine + ((c - half) * 8 + k) * kPRows;
                const float4 old = __ldcg(to);
                *to = make_float4(old.x * fa, old.y * fa, old.z * fa, old.w * fa);
            }
    }
    if (first || rebase) *base = make_float2(ref, __int_as_float(top_scale));
    __syncwarp();                                      /* rows of a warp differ in that; what follows takes all of them together */
#pragma unroll 1
    for (int c = half; c < NB; c += 2) {
        uint32_t reg[32];
        at_ld32(tO + (uint32_t)(c * 32), reg);
        float4 *to = mine + (c - half) * 8 * kPRows;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const float4 v = make_float4(__uint_as_float(reg[4 * k]) * g, __uint_as_float(reg[4 * k + 1]) * g, __uint_as_float(reg[4 * k + 2]) * g,
                                         __uint_as_float(reg[4 * k + 3]) * g);
            if (first) to[k * kPRows] = v;
            else atomicAdd(to + k * kPRows, v);        /* this thread alone adds here, so in one order */
        }
    }
}

/* Scales too far apart: all that this CTA has, in fp32, over what was left by then. By itself, with arguments by value and places worked out
 * again, so that nothing is kept for it in the kernel's registers (1203 rows: 212 us so, 211 now). */
template <int NB, class T>
__device__ __noinline__ void p_plain(const Kv4Attn a, const ServeRows<T> q, const ServeRows<T> out) {
    constexpr int kDim = NB * 32, kPart = kPRows * (kDim + 2);
    extern __shared__ unsigned char p_smem_raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float *q_row = reinterpret_cast<float *>(((uintptr_t)p_smem_raw + 1023) & ~(uintptr_t)1023) + warp * 2 * kDim, *results = q_row + kDim;
    PWork work;
    p_work(a, blockIdx.x, work);
    const Kv4Head cache = kv4_head<NB>(a.c, a.c.row(work.seq, work.kv_head, 0));
    float *part = a.part + (size_t)work.slot * kPart;
    for (int p = warp; p < work.n_pairs; p += kPThreads / 32) {
        const int row = (work.pair0 + p) / a.group, head = work.kv_head * a.group + work.pair0 + p - row * a.group;
        const float2 end = kv4_plain_row<NB, T>(cache, q.data + work.seq * q.seq + row * q.row + head * q.head, a.scale, work.first_tile * kPKeys,
                                                min((work.first_tile + work.n_tiles) * kPKeys, work.before + row + 1), q_row, results);
        const float inv = end.y == 0.0f ? 0.0f : 1.0f / end.y;
        for (int d = lane; d < kDim; d += 32) {
            if (work.used > 1) part[p * kDim + d] = results[d];
            else serve_put(out.data + work.seq * out.seq + row * out.row + head * out.head + d, end.y == 0.0f ? 0.0f : results[d] * inv);
        }
        if (lane == 0) {
            if (work.used > 1) reinterpret_cast<float2 *>(part + kPRows * kDim)[p] = end;
            else if (a.lse) a.lse[((size_t)work.seq * a.max_rows + row) * a.heads + head] = end.y == 0.0f ? -INFINITY : (end.x + (float)kKv4Rest + log2f(end.y)) * 0.69314718f;
        }
        __syncwarp();
    }
}

template <int NB, int PT, class T>
__global__ void __launch_bounds__(kPThreads, 1) kv4_prompt_kernel(const Kv4Attn a, const ServeRows<T> q, const ServeRows<T> out) {
    constexpr int QT = sizeof(T) == 4 ? 2 : 1, kDim = NB * 32;
    using Cfg = PCfg<NB, QT>;
    extern __shared__ unsigned char p_smem_raw[];
    unsigned char *base = (unsigned char *)(((uintptr_t)p_smem_raw + 1023) & ~(uintptr_t)1023);
    unsigned char *q_s = base, *k_s = q_s + Cfg::kQ, *v_s = k_s + Cfg::kSlots * Cfg::kSlot;
    __shared__ __align__(8) uint64_t k_full[Cfg::kSlots], k_empty[Cfg::kSlots], v_full[Cfg::kSlots], v_empty[Cfg::kSlots], s_full[2], p_full[2], o_done[2], q_full;
    __shared__ float key_up[kPRing][4], down_s[kPRows], top_s[2][2][kPRows];
    __shared__ float2 aside_s[2][2][kPRows];                       /* reference, scale of what is put aside */
    __shared__ int value_top[kPRing], bad_s[NB], abort_s, room_s, far_s;
    __shared__ uint32_t tmem_slot;
    int *abort_flag = &abort_s;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    PWork work;
    if (!p_work(a, blockIdx.x, work)) return;
    const int seq = work.seq, kv_head = work.kv_head, pair0 = work.pair0, n_pairs = work.n_pairs, pairs = pair0 + n_pairs, before = work.before, seen = work.seen;
    const int first_tile = work.first_tile, n_tiles = work.n_tiles, used = work.used;
    const int all_see = before + pair0 / a.group + 1;
    if (tid == 0) {
        for (int i = 0; i < Cfg::kSlots; i++) {
            vb_mbar_init(&k_full[i], 4);
            vb_mbar_init(&v_full[i], 4);
            vb_mbar_init(&k_empty[i], 1);
            vb_mbar_init(&v_empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            vb_mbar_init(&s_full[i], 1);
            vb_mbar_init(&p_full[i], 256);
            vb_mbar_init(&o_done[i], 1);
        }
        vb_mbar_init(&q_full, kPSoft);
        abort_s = far_s = 0;
        vb_mbar_init_fence();
    }
    if (tid < NB) bad_s[tid] = 1 << 30;
    const bool puts_aside = n_tiles > 2 * Cfg::kChain;
    if (puts_aside && tid == 32) {
        int room;
        if (!p_take(a, room)) atomicCAS(a.status, 0, kPStatus);
        room_s = room;
    }
    if (warp == kPMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(vb_smem_u32(&tmem_slot)), "r"(kPTmem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();       /* not before the allocation: a kernel that starts early must not take columns this one needs */
    const uint32_t tmem = *(volatile uint32_t *)&tmem_slot;
    auto give_up = [&]() {
        atomicCAS(a.status, 0, kPStatus);
        *(volatile int *)abort_flag = 1;
    };

    if (warp < kPSoft / 32) {
        /* ---- queries: four values a lane, NB * 8 lanes a row, so that a warp has one, two or four rows at a time; the loads of
         * its eight rows together ---- */
        constexpr int kLanes = NB * 8, kSide = 32 / kLanes, kBatch = 8 / kSide;
        const int side = lane / kLanes, d = (lane - side * kLanes) * 4;
        const bool mine = side < kSide;
        ServeRaw4<T> raw[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; u++) {
            const int pair = pair0 + warp * 8 + u * kSide + side;
            const bool real = mine && pair < pairs;
            const int row = real ? pair / a.group : 0, head = kv_head * a.group + (real ? pair - row * a.group : 0);
            const T *p = q.data + seq * q.seq + row * q.row + head * q.head + d;
            raw[u].none();
            if (real) raw[u].load(p, a.wide);
        }
#pragma unroll
        for (int u = 0; u < kBatch; u++) {
            const int r = warp * 8 + u * kSide + side;
            const float4 x = raw[u].get();
            uint32_t most = max(max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu), max(__float_as_uint(x.z) & 0x7fffffffu, __float_as_uint(x.w) & 0x7fffffffu));
            if constexpr (kSide == 1) {
                most = __reduce_max_sync(0xffffffffu, most);
            } else {
#pragma unroll
                for (int o = 1; o < kLanes; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
            }
            const uint32_t e = most >> 23, field = e == 0u || e == 255u ? 127u : min(268u - e, 253u);
            float up = __uint_as_float(field << 23);
            if (mine && d == 0) down_s[r] = __uint_as_float((254u - field) << 23);
            if (a.scale <= 0.0f) up = a.scale < 0.0f ? -up : 0.0f;      /* the largest score is the largest product */
            if (mine) {
                const uint32_t at = (uint32_t)(d >> 6) * kPBlock + at_off(r, (d & 63) >> 3) + (d & 7) * 2;
                const float y0 = x.x * up, y1 = x.y * up, y2 = x.z * up, y3 = x.w * up;
                const uint2 hi = make_uint2(half_pack(y0, y1), half_pack(y2, y3));
                *reinterpret_cast<uint2 *>(q_s + at) = hi;
                if constexpr (QT == 2) {
                    const float2 f = kv4_f2(hi.x), g = kv4_f2(hi.y);
                    *reinterpret_cast<uint2 *>(q_s + Cfg::kSlot + at) = make_uint2(half_pack(y0 - f.x, y1 - f.y), half_pack(y2 - g.x, y3 - g.y));
                }
            }
        }
        at_proxy_fence();
        vb_mbar_arrive(&q_full);
        vb_named_bar(1, kPSoft);                                   /* down_s */

        /* ---- softmax: two warpgroups take tiles w, w + 2, ...; a thread has half of the columns of pair pair0 + r ---- */
        const int wg = warp >> 2, w = wg >> 1, half = wg & 1, r = tid & 127, pair = pair0 + r;
        const bool valid = r < n_pairs;
        const int row = valid ? pair / a.group : 0, head = kv_head * a.group + (valid ? pair - row * a.group : 0);
        const int sees = before + (pair0 + min(r, n_pairs - 1)) / a.group + 1;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, tS = tmem + lanes + (uint32_t)(w * kPKeys), tO = tmem + lanes + kPO + (uint32_t)(w * 128);
        /* positive, so that what is masked stays -inf: queries are zeros where the scale is */
        const float mul = (a.scale != 0.0f ? fabsf(a.scale) * 1.44269504f : 1.0f) * down_s[r];
        float ref = -INFINITY, sum = 0.0f;
        int top_scale = 0, it = 0, t = w;
        for (; t < n_tiles; t += 2, it++) {
            const int j0 = (first_tile + t) * kPKeys;
            if (!at_warp_wait(&s_full[w], (uint32_t)it & 1u, abort_flag)) { give_up(); break; }
            tc_fence_after();
            /* the products up to it - 1 were done before these scores were begun; the next starts from zero */
            if (it > 0 && it % Cfg::kChain == 0)
                p_put_aside<NB>(p_aside<NB>(a, *(volatile int *)&room_s, w, half) + r, &aside_s[w][half][r], tO, half, it == Cfg::kChain, ref, top_scale);
            const float *ups = key_up[t % kPRing];
            const int last = sees - j0;                            /* columns before this one are seen */
            const bool masked = j0 + kPKeys > all_see;
            float top = -INFINITY;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                uint32_t reg[32];
                const int column = half * 64 + c * 32;
                at_ld32(tS + (uint32_t)column, reg);
                if (masked) {
#pragma unroll
                    for (int k = 0; k < 32; k++)
                        if (column + k >= last) reg[k] = 0xff800000u;
                }
                float m4[4];
#pragma unroll
                for (int k = 0; k < 4; k++) m4[k] = __uint_as_float(reg[k]);
#pragma unroll
                for (int k = 4; k < 32; k++) m4[k & 3] = fmaxf(m4[k & 3], __uint_as_float(reg[k]));
                const float m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                top = m > -INFINITY ? fmaxf(top, m * (ups[half * 2 + c] * mul)) : top;
                __syncwarp();                          /* lanes are together where the next columns are read */
            }
            /* the other half's: it has been read by then when it is written again, since the next tile's scores wait for both halves */
            top_s[w][half][r] = top;
            vb_named_bar(2 + w, 256);
            top = fmaxf(top, top_s[w][half ^ 1][r]);
            /* values: the scale that this tile is based on */
            if (!at_warp_wait(&v_full[t % Cfg::kSlots], (uint32_t)(t / Cfg::kSlots) & 1u, abort_flag)) { give_up(); t += 2; break; }
            const int now_scale = value_top[t % kPRing];
            const bool rise = top > ref + kPTrail;
            if (__any_sync(0xffffffffu, rise) || now_scale != top_scale) {
                const float now = rise ? top : ref, f = rise ? exp2_fast(ref - now) : 1.0f;      /* the first time: 0 */
                if (it > 0) {
                    if (!at_warp_wait(&o_done[w], (uint32_t)(it - 1) & 1u, abort_flag)) { give_up(); t += 2; break; }
                    tc_fence_after();
                    const int fall = now_scale - top_scale;
                    const float fo = fall > 126 ? 0.0f : f * __uint_as_float((uint32_t)(127 - fall) << 23);
#pragma unroll 1
                    for (int c = half; c < NB; c += 2) {
                        uint32_t reg[32];
                        at_ld32(tO + (uint32_t)(c * 32), reg);
#pragma unroll
                        for (int k = 0; k < 32; k++) reg[k] = __float_as_uint(__uint_as_float(reg[k]) * fo);
                        at_st32(tO + (uint32_t)(c * 32), reg);
                    }
                }
                sum *= f;
                ref = now;
                top_scale = now_scale;
            }
            const float low = ref > -INFINITY ? ref - kPBias : 0.0f;      /* nothing seen yet: every weight is 2^-inf */
            uint64_t sums[2] = {0, 0};
            const uint64_t low2 = vb_f2_pack(-low, -low);
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int column = half * 64 + c * 32;
                const float up = fmaxf(ups[half * 2 + c] * mul, 0x1p-149f);      /* not 0, whatever the scales: what is masked stays -inf */
                const uint64_t up2 = vb_f2_pack(up, up);
                uint32_t s[32], second[PT == 2 ? 16 : 1];
                at_ld32(tS + (uint32_t)column, s);
                if (masked) {
#pragma unroll
                    for (int k = 0; k < 32; k++)
                        if (column + k >= last) s[k] = 0xff800000u;
                }
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    const float2 x = vb_f2_get(vb_f2_fma(vb_f2_pack(__uint_as_float(s[k]), __uint_as_float(s[k + 1])), up2, low2));
                    const float p0 = exp2_fast(x.x), p1 = exp2_fast(x.y);
                    sums[(k >> 1) & 1] = vb_f2_add(sums[(k >> 1) & 1], vb_f2_pack(p0, p1));
                    const uint32_t hi = half_pack(p0, p1);
                    s[k / 2] = hi;
                    if constexpr (PT == 2) {
                        const float2 f = kv4_f2(hi);
                        second[k / 2] = half_pack(p0 - f.x, p1 - f.y);
                    }
                }
                p_st16(tS + (uint32_t)column, s);                  /* 16 columns of first terms, 16 of second ones */
                if constexpr (PT == 2) p_st16(tS + (uint32_t)(column + 16), second);
            }
            const float2 sum2 = vb_f2_get(vb_f2_add(sums[0], sums[1]));
            sum += sum2.x + sum2.y;
            at_st_wait();
            tc_fence_before();
            vb_mbar_arrive(&p_full[w]);
        }
        for (; t < n_tiles; t += 2) vb_named_bar(2 + w, 256);         /* given up: the others of the pair meet its barrier all the same */
        if (it > 0 && !at_warp_wait(&o_done[w], (uint32_t)(it - 1) & 1u, abort_flag)) give_up();
        /* the tiles of either pair of warpgroups, merged, a warpgroup a block of 32 columns, by way of shared memory */
        vb_named_bar(1, kPSoft);                                     /* every product is done: the rings are free */
        float4 *ends = reinterpret_cast<float4 *>(k_s);            /* 4 x 128 x (reference, sum, scale) */
        float *rows = reinterpret_cast<float *>(k_s + 4 * kPRows * 16);
        ends[wg * kPRows + r] = make_float4(ref, sum * kPOut, __int_as_float(top_scale), 0.0f);
        if (puts_aside) __threadfence();
        tc_fence_before();
        vb_named_bar(1, kPSoft);
        tc_fence_after();
        float4 A = ends[r], B = ends[2 * kPRows + r];
        A.y += ends[kPRows + r].y;
        B.y += ends[3 * kPRows + r].y;
        const float reference = fmaxf(A.x, B.x);
        float fa = A.x > -INFINITY ? exp2_fast(A.x - reference) : 0.0f, fb = B.x > -INFINITY ? exp2_fast(B.x - reference) : 0.0f;
        const float total = A.y * fa + B.y * fb, inv = used > 1 ? 1.0f : total == 0.0f ? 0.0f : 1.0f / total;
        float *part = a.part + (size_t)work.slot * PCfg<NB, QT>::kPart;
        if (used > 1) {
            if (wg == 0) reinterpret_cast<float2 *>(part + kPRows * kDim)[r] = make_float2(reference, total);
        } else if (wg == 0 && valid && a.lse)
            a.lse[((size_t)seq * a.max_rows + row) * a.heads + head] = total == 0.0f ? -INFINITY : (reference + (float)kKv4Rest + log2f(total)) * 0.69314718f;
        fa *= inv;
        fb *= inv;
        const int ea = __float_as_int(A.z) - kPDown, eb = __float_as_int(B.z) - kPDown;      /* in two steps: 2^e may not be a normal number */
        const float a0 = __uint_as_float((uint32_t)(127 + (ea >> 1)) << 23), a1 = __uint_as_float((uint32_t)(127 + ea - (ea >> 1)) << 23);
        const float b0 = __uint_as_float((uint32_t)(127 + (eb >> 1)) << 23), b1 = __uint_as_float((uint32_t)(127 + eb - (eb >> 1)) << 23);
#pragma unroll 1
        for (int c = wg; c < NB; c += kPSoft / 128) {
            uint32_t oa[32], ob[32];
            const bool nan = bad_s[c] < sees;
            __syncwarp();
            if (n_tiles > 0) at_ld32(tmem + lanes + kPO + (uint32_t)(c * 32), oa);
            if (n_tiles > 1) at_ld32(tmem + lanes + kPO + 128u + (uint32_t)(c * 32), ob);
#pragma unroll
            for (int k = 0; k < 32; k++) {
                float v = 0.0f;
                if (n_tiles > 0) v = __uint_as_float(oa[k]) * a0 * fa * a1;
                if (n_tiles > 1) v += __uint_as_float(ob[k]) * b0 * fb * b1;
                oa[k] = __float_as_uint(v);
            }
#pragma unroll 1
            for (int x = 0; x < 2 && n_tiles > 2 * Cfg::kChain + x; x++) {
                const float2 e = aside_s[x][0][r];
                const int scale = __float_as_int(e.y) - kPDown;
                const float f = e.x > -INFINITY ? exp2_fast(e.x - reference) * inv : 0.0f;
                const float s0 = __uint_as_float((uint32_t)(127 + (scale >> 1)) << 23), s1 = __uint_as_float((uint32_t)(127 + scale - (scale >> 1)) << 23);
                const float4 *from = p_aside<NB>(a, room_s, x, c) + r;
#pragma unroll
                for (int k = 0; k < 32; k += 4) {
                    const float4 o = __ldcg(from + k / 4 * kPRows);
                    oa[k] = __float_as_uint(__uint_as_float(oa[k]) + o.x * s0 * f * s1);
                    oa[k + 1] = __float_as_uint(__uint_as_float(oa[k + 1]) + o.y * s0 * f * s1);
                    oa[k + 2] = __float_as_uint(__uint_as_float(oa[k + 2]) + o.z * s0 * f * s1);
                    oa[k + 3] = __float_as_uint(__uint_as_float(oa[k + 3]) + o.w * s0 * f * s1);
                }
            }
#pragma unroll
            for (int k = 0; k < 32; k++) {
                if (total == 0.0f) oa[k] = 0u;                     /* nothing seen */
                if (nan) oa[k] = 0x7fffffffu;
            }
#pragma unroll
            for (int k = 0; k < 32; k += 4) *reinterpret_cast<uint4 *>(rows + r * Cfg::kLd + c * 32 + k) = make_uint4(oa[k], oa[k + 1], oa[k + 2], oa[k + 3]);
        }
        vb_named_bar(1, kPSoft);
        /* out, eight values a lane */
        constexpr int kEights = kDim / 8;
        for (int x = tid; x < n_pairs * kEights; x += kPSoft) {
            const int p = x / kEights, d = (x - p * kEights) * 8, rr = (pair0 + p) / a.group, hh = kv_head * a.group + pair0 + p - rr * a.group;
            const float4 lo = *reinterpret_cast<const float4 *>(rows + p * Cfg::kLd + d), hi = *reinterpret_cast<const float4 *>(rows + p * Cfg::kLd + d + 4);
            if (used > 1) {
                reinterpret_cast<float4 *>(part + p * kDim + d)[0] = lo;
                reinterpret_cast<float4 *>(part + p * kDim + d)[1] = hi;
                continue;
            }
            const float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
            serve_store<8>(out.data + seq * out.seq + rr * out.row + hh * out.head + d, a.wide_out, v);
        }
    } else if (warp < 20) {
        /* ---- keys: a warp has 32 tokens of a tile, four lanes a token (words t * NB ..: values 8 t .. of every block) ---- */
        const int lw = warp - 16, g = lane >> 2, tq = lane & 3;
        const size_t row0 = a.c.row(seq, kv_head, 0);
        uint32_t words[4][NB], bytes[4][NB];
        auto fetch = [&](int t) {
            const int j0 = (first_tile + t) * kPKeys, end = a.c.slots - 1 - j0;             /* slots are whole tiles of 64: half of the last 128 may be none */
            const unsigned char *codes = a.c.k + (row0 + j0) * (NB * 16), *scales = a.c.ks + (row0 + j0) * NB;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int r = min(lw * 32 + i * 8 + g, end);
                get_words<NB>(codes + r * (NB * 16) + tq * (NB * 4), words[i]);
                get_bytes<NB>(scales + r * NB, bytes[i]);
            }
        };
        if (n_tiles > 0) fetch(0);
        for (int t = 0; t < n_tiles; t++) {
            const int slot = t % Cfg::kSlots, j0 = (first_tile + t) * kPKeys + lw * 32;
            int most = 0;
            uint32_t least = 255u;                     /* less one: zeros, which nothing is lost of, come last */
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    if (j0 + i * 8 + g >= seen) { words[i][b] = 0; bytes[i][b] = 0; }       /* whatever lies behind the last token */
                }
            /* four lanes have the same tokens: each looks at one of them */
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const uint32_t byte = tq < 2 ? (tq == 0 ? bytes[0][b] : bytes[1][b]) : tq == 2 ? bytes[2][b] : bytes[3][b];
                if (byte != 255u) most = max(most, (int)byte);
                least = min(least, byte - 1u);
            }
            most = max((int)__reduce_max_sync(0xffffffffu, (unsigned)most), 14);          /* its undoing stays a normal number */
            if (kv4_far(least + 1u, most)) *(volatile int *)&far_s = 1;
            if (!at_warp_wait(&k_empty[slot], ((uint32_t)(t / Cfg::kSlots) & 1u) ^ 1u, abort_flag)) { give_up(); break; }
            unsigned char *to = k_s + slot * Cfg::kSlot;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int r = lw * 32 + i * 8 + g;
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    uint4 v = p_halves(words[i][b], p_factor((int)bytes[i][b], most));
                    if (bytes[i][b] == 255u) v.x = 0x7fff7fffu;            /* a block that is NaN: so is the score */
                    const int chunk = 4 * b + tq;
                    *reinterpret_cast<uint4 *>(to + (chunk >> 3) * kPBlock + at_off(r, chunk & 7)) = v;
                }
            }
            if (lane == 0) key_up[t % kPRing][lw] = __uint_as_float((uint32_t)(most - 13) << 23);
            if (t + 1 < n_tiles) fetch(t + 1);
            at_proxy_fence();
            __syncwarp();
            if (lane == 0) vb_mbar_arrive(&k_full[slot]);
        }
    } else if (warp < kPMmaWarp) {
        /* ---- values: the warps take 32 tokens in turn, a lane blocks of them ---- */
        const size_t row0 = a.c.row(seq, kv_head, 0);
        uint32_t words[NB][4], byte[NB], all[NB];
        auto fetch = [&](int task) {
            const int j0 = (first_tile + task / 4) * kPKeys, end = a.c.slots - 1 - j0;          /* slots are whole tiles of 64: half of the last 128 may be none */
            const unsigned char *codes = a.c.v + (row0 + j0) * (NB * 16), *scales = a.c.vs + (row0 + j0) * NB;
#pragma unroll
            for (int i = 0; i < NB; i++) {
                const int x = i * 32 + lane, key = x / NB, b = x - key * NB, r = min(task % 4 * 32 + key, end);
                if constexpr (kv4_whole(NB)) {
                    get_words<4>(codes + r * (NB * 16) + b * 16, words[i]);
                } else {
                    const uint16_t *h = reinterpret_cast<const uint16_t *>(codes + r * (NB * 16)) + b;
#pragma unroll
                    for (int k = 0; k < 4; k++) words[i][k] = h[2 * k * NB] | ((uint32_t)h[(2 * k + 1) * NB] << 16);
                }
                byte[i] = scales[r * NB + b];
            }
            /* all scales of the tile, four tokens a lane: every warp finds the largest for itself */
            const uint32_t *four = reinterpret_cast<const uint32_t *>(scales + min(lane * 4, end - 3) * NB);
#pragma unroll
            for (int i = 0; i < NB; i++) all[i] = four[i];
        };
        int top = 0, first_top = 0;
        const int tasks = n_tiles * 4;
        if (warp - 20 < tasks) fetch(warp - 20);
        for (int task = warp - 20; task < tasks; task += 3) {
            const int t = task / 4, lw = task % 4, slot = t % Cfg::kSlots, j0 = (first_tile + t) * kPKeys;
            const int real = seen - j0;                            /* tokens of the tile that are seen */
            /* the largest and the smallest byte of the tile, two at a time; by themselves where some do not count */
            uint32_t hi = 0u, lo = 0x00ff00ffu;
#pragma unroll
            for (int i = 0; i < NB; i++) {
                const uint32_t even = all[i] & 0x00ff00ffu, odd = (all[i] >> 8) & 0x00ff00ffu;
                hi = __vmaxu2(hi, __vmaxu2(even, odd));
                lo = __vminu2(lo, __vminu2(even, odd));
            }
            int most = (int)max(hi & 0xffffu, hi >> 16);
            uint32_t least = min(lo & 0xffffu, lo >> 16);
            if (__any_sync(0xffffffffu, real < kPKeys || most == 255 || least == 0u)) {
                most = 0;
                least = 255u;
#pragma unroll
                for (int i = 0; i < NB * 4; i++) {
                    const uint32_t byte_i = (all[i / 4] >> (8 * (i % 4))) & 255u;
                    if (lane * 4 + i / NB >= real) continue;
                    if (byte_i == 255u) atomicMin(&bad_s[i % NB], j0 + lane * 4 + i / NB);      /* a block that is NaN: the rows that see it; its codes are zeros */
                    else most = max(most, (int)byte_i);
                    least = min(least, byte_i - 1u);       /* zeros, which nothing is lost of, come last */
                }
                least = least < 254u ? least + 1u : 255u;
                __syncwarp();
            }
            top = max(top, (int)__reduce_max_sync(0xffffffffu, (unsigned)most));
            if (first_top == 0) first_top = top;
            if (kv4_far(least, top) || top - first_top > kKv4Rise) *(volatile int *)&far_s = 1;
            if (!at_warp_wait(&v_empty[slot], ((uint32_t)(t / Cfg::kSlots) & 1u) ^ 1u, abort_flag)) { give_up(); break; }
            unsigned char *to = v_s + slot * Cfg::kSlot;
#pragma unroll
            for (int i = 0; i < NB; i++) {
                const int x = i * 32 + lane, key = x / NB, b = x - key * NB, r = lw * 32 + key;
                const bool none = r >= real || byte[i] == 255u;
                const uint32_t f = none ? 0u : p_factor((int)byte[i], top);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int chunk = 4 * b + k;
                    *reinterpret_cast<uint4 *>(to + (chunk >> 3) * kPBlock + at_off(r, chunk & 7)) = p_halves(none ? 0u : words[i][k], f);
                }
            }
            if (lw == 0 && lane == 0) value_top[t % kPRing] = top;
            if (task + 3 < tasks) fetch(task + 3);
            at_proxy_fence();
            __syncwarp();
            if (lane == 0) vb_mbar_arrive(&v_full[slot]);
        }
    } else if (lane == 0) {
        /* ---- MMA issuer ---- */
        const uint32_t idesc_s = p_idesc(kPKeys, false), idesc_o = p_idesc(kDim, true);
        const AtDesc k_desc(umma_desc_k_sw128(k_s)), q_desc(umma_desc_k_sw128(q_s)), v_desc(p_desc_mn(vb_smem_u32(v_s)));
        bool ok = vb_mbar_wait(&q_full, 0u, abort_flag);
        tc_fence_after();
        auto scores = [&](int t) {
            const int slot = t % Cfg::kSlots;
            if (!vb_mbar_wait(&k_full[slot], (uint32_t)(t / Cfg::kSlots) & 1u, abort_flag)) return false;
            tc_fence_after();
            const AtDesc kd = k_desc.at(slot * (Cfg::kSlot >> 4));
            const uint32_t d = tmem + (uint32_t)((t & 1) * kPKeys);
#pragma unroll
            for (int ks = 0; ks < NB * 2; ks++) {
                const int at = (ks >> 2) * (kPBlock >> 4) + 2 * (ks & 3);
#pragma unroll
                for (int u = 0; u < QT; u++) at_mma_ss(d, q_desc.at(at + u * (Cfg::kSlot >> 4)), kd.at(at), idesc_s, ks + u != 0 ? 1u : 0u);
            }
            umma_commit(&k_empty[slot]);
            umma_commit(&s_full[t & 1]);
            return true;
        };
        ok = ok && n_tiles > 0 && scores(0);
        if (ok && n_tiles > 1) ok = scores(1);
        for (int t = 0; t < n_tiles && ok; t++) {
            const int w = t & 1, slot = t % Cfg::kSlots;
            ok = vb_mbar_wait(&v_full[slot], (uint32_t)(t / Cfg::kSlots) & 1u, abort_flag) && vb_mbar_wait(&p_full[w], (uint32_t)(t >> 1) & 1u, abort_flag);
            if (!ok) break;
            tc_fence_after();
            const AtDesc vd = v_desc.at(slot * (Cfg::kSlot >> 4));
            const uint32_t d = tmem + kPO + (uint32_t)(w * 128);
#pragma unroll
            for (int ks = 0; ks < kPKeys / 16; ks++) {
                const uint32_t p = tmem + (uint32_t)(w * kPKeys + (ks >> 1) * 32 + (ks & 1) * 8);
#pragma unroll
                for (int u = 0; u < PT; u++) at_mma_ts(d, p + u * 16, vd.at(ks * (2048 >> 4)), idesc_o, ((t >> 1) % Cfg::kChain | ks | u) != 0 ? 1u : 0u);
            }
            umma_commit(&v_empty[slot]);
            umma_commit(&o_done[w]);
            /* takes the columns of P once the products above have read them: MMAs of one thread run in order */
            if (t + 2 < n_tiles) ok = scores(t + 2);
        }
        if (!ok && n_tiles > 0) give_up();
    }
    tc_fence_before();
    __syncthreads();
    if (*(volatile int *)&far_s) p_plain<NB, T>(a, q, out);
    if (puts_aside && tid == 32) {
        __threadfence();
        atomicExch(&a.rooms[room_s], 0u);
    }
    if (warp == kPMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kPTmem) : "memory");
    }
}

/* The parts of cut sequences together: a CTA takes a share of the rows of the unit that the CTA of its number had a part of, a warp a row. */
constexpr int kJThreads = 256;
template <int NB, class T>
__global__ void __launch_bounds__(kJThreads) kv4_join_kernel(const Kv4Attn a, const ServeRows<T> out) {
    constexpr int kDim = NB * 32, kPart = kPRows * (kDim + 2);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    PWork work;
    if (!p_work(a, blockIdx.x + (a.split ? 0 : a.tail0), work) || work.used == 1) return;
    const int seq = work.seq, kv_head = work.kv_head, pair0 = work.pair0, n_pairs = work.n_pairs, used = work.used, split = work.split;
    const float *parts = a.part + (size_t)(work.slot - split * work.stride) * kPart;
    const size_t step = (size_t)work.stride * kPart;
    for (int p = split + warp * used; p < n_pairs; p += kJThreads / 32 * used) {
        auto end = [&](int x) { return __ldcg(reinterpret_cast<const float2 *>(parts + x * step + kPRows * kDim) + p); };
        float reference = -INFINITY, total = 0.0f;
        for (int x = lane; x < used; x += 32) reference = fmaxf(reference, end(x).x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) reference = fmaxf(reference, __shfl_xor_sync(0xffffffffu, reference, o));
        float v[NB];
#pragma unroll
        for (int i = 0; i < NB; i++) v[i] = 0.0f;
        for (int x0 = 0; x0 < used; x0 += 32) {
            const float2 e = x0 + lane < used ? end(x0 + lane) : make_float2(-INFINITY, 0.0f);
            const float mine = e.x > -INFINITY ? exp2_fast(e.x - reference) : 0.0f;
            float sum = e.y * mine;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            total += sum;
            const int n = min(32, used - x0);
#pragma unroll 4
            for (int x = 0; x < n; x++) {
                const float f = __shfl_sync(0xffffffffu, mine, x);
                const float *row = parts + (x0 + x) * step + p * kDim + lane * NB;
#pragma unroll
                for (int i = 0; i < NB; i++) v[i] = fmaf(__ldcg(row + i), f, v[i]);
            }
        }
        const int pair = pair0 + p, row = pair / a.group, head = kv_head * a.group + pair - row * a.group;
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        T *to = out.data + seq * out.seq + row * out.row + head * out.head + lane * NB;
#pragma unroll
        for (int i = 0; i < NB; i++) serve_put(to + i, total == 0.0f ? 0.0f : v[i] * inv);
        if (lane == 0 && a.lse) a.lse[((size_t)seq * a.max_rows + row) * a.heads + head] = total == 0.0f ? -INFINITY : (reference + (float)kKv4Rest + log2f(total)) * 0.69314718f;
    }
}

/* ------------------------------------------------------------------ the weight of each token, for many rows
 *   S^T [128 tokens x 128 pairs] = K Q^T,  mass_j = sum over pairs of exp(S_j - lse), a thread per token
 * A CTA has 128 tokens of a KV head, whose keys stay in shared memory; the pairs that see them come by 128 at a time: eight warps bring
 * queries to FP16, one issues the products, two warpgroups take alternate tiles of pairs. A token's weights are summed in one order.
 * 1024 rows of 32 heads over 4096 tokens, 256 CTAs on 148 SMs: 197 us by itself (840 on warp-level MMAs, whose keys are decoded again for every
 * eight pairs), issue slots 58 % busy, the tensor pipe 9: every CTA brings the queries to FP16 again, and eight warps take the exponentials. */
constexpr int kWMmaWarp = 16, kWThreads = 32 * (kWMmaWarp + 1), kWSlots = 2, kWStatus = 63, kWRing = 4;
constexpr uint32_t kWTmem = 256;

template <int NB, int QT>
struct WCfg {
    static constexpr int kSlot = (NB + 1) / 2 * kPBlock;
    static constexpr int kSmem = kSlot + kWSlots * QT * kSlot + 1024;
};

template <int NB, class T>
__global__ void __launch_bounds__(kWThreads, 1) kv4_mass_many_kernel(const Kv4Attn a, const ServeRows<T> q) {
    constexpr int QT = sizeof(T) == 4 ? 2 : 1;
    using Cfg = WCfg<NB, QT>;
    extern __shared__ unsigned char p_smem_raw[];
    unsigned char *base = (unsigned char *)(((uintptr_t)p_smem_raw + 1023) & ~(uintptr_t)1023);
    unsigned char *k_s = base, *q_s = k_s + Cfg::kSlot;
    __shared__ __align__(8) uint64_t q_full[kWSlots], q_empty[kWSlots], s_full[2], s_empty[2], k_full;
    __shared__ __align__(16) float2 pair_s[kWRing][kPRows];                 /* of a pair: what S is multiplied by, its lse in powers of two */
    __shared__ float sum_s[kPKeys];
    __shared__ int abort_s, far_s;
    __shared__ uint32_t tmem_slot;
    int *abort_flag = &abort_s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, kv_head = blockIdx.y, seq = blockIdx.z, tok0 = blockIdx.x * kPKeys;
    /* begins beside the end of the attention's kernels, which have waited for all that is read here but lse; masses may not be written
     * before those are waited for either */
    const Kv4Span span = kv4_span(a.lengths, a.rows, a.max_rows, seq, a.c.capacity);
    const int pairs = span.rows * a.group, before = span.length - span.rows;
    if (tok0 >= span.length) {
        pdl_wait();                /* no launch is over before the ones it follows are */
        return;
    }
    /* rows before this CTA's first token see none of its tokens */
    const int first = (int)min((long long)pairs, (long long)max(0, tok0 - before) * a.group) / kPRows * kPRows, n_tiles = (pairs - first + kPRows - 1) / kPRows;
    if (tid == 0) {
        for (int i = 0; i < kWSlots; i++) {
            vb_mbar_init(&q_full[i], 8);
            vb_mbar_init(&q_empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            vb_mbar_init(&s_full[i], 1);
            vb_mbar_init(&s_empty[i], 128);
        }
        vb_mbar_init(&k_full, 8);
        abort_s = far_s = 0;
        vb_mbar_init_fence();
    }
    if (warp == kWMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(vb_smem_u32(&tmem_slot)), "r"(kWTmem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *(volatile uint32_t *)&tmem_slot;
    auto give_up = [&]() {
        atomicCAS(a.status, 0, kWStatus);
        *(volatile int *)abort_flag = 1;
    };

    if (warp < 8) {
        /* ---- keys: a warp has 16 tokens, four lanes a token; a token's scales against the largest of its 16 ---- */
        const int g = lane >> 2, tq = lane & 3;
        const size_t row0 = a.c.row(seq, kv_head, 0);
        __shared__ float key_up[8];
        uint32_t words[2][NB], bytes[2][NB], least = 255u;
        int most = 0;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int j = tok0 + warp * 16 + i * 8 + g;
            const size_t row = row0 + min(j, a.c.slots - 1);
            get_words<NB>(a.c.k + row * (NB * 16) + tq * (NB * 4), words[i]);
            get_bytes<NB>(a.c.ks + row * NB, bytes[i]);
#pragma unroll
            for (int b = 0; b < NB; b++) {
                if (j >= span.length) { words[i][b] = 0; bytes[i][b] = 0; }
                if (bytes[i][b] != 255u) most = max(most, (int)bytes[i][b]);
                least = min(least, bytes[i][b] - 1u);
            }
        }
        most = max((int)__reduce_max_sync(0xffffffffu, (unsigned)most), 14);              /* its undoing stays a normal number */
        if (kv4_far(least + 1u, most)) *(volatile int *)&far_s = 1;
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int b = 0; b < NB; b++) {
                uint4 v = p_halves(words[i][b], p_factor((int)bytes[i][b], most));
                if (bytes[i][b] == 255u) v.x = 0x7fff7fffu;                /* a block that is NaN: so is the score */
                const int chunk = 4 * b + tq;
                *reinterpret_cast<uint4 *>(k_s + (chunk >> 3) * kPBlock + at_off(warp * 16 + i * 8 + g, chunk & 7)) = v;
            }
        if (lane == 0) key_up[warp] = __uint_as_float((uint32_t)(most - 13) << 23);
        at_proxy_fence();
        __syncwarp();
        if (lane == 0) vb_mbar_arrive(&k_full);
        vb_named_bar(1, 256);

        /* ---- sums: warpgroup w takes tiles w, w + 2, ... of pairs, a thread token tok0 + r ---- */
        const int w = warp >> 2, r = tid & 127, j = tok0 + r;
        const uint32_t tS = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(w * kPRows);
        pdl_wait();                                                        /* bounded waits begin when the kernels before are done, however long they take */
        const float up = key_up[r >> 4];
        const uint64_t up2 = vb_f2_pack(up, up);
        uint64_t sums[2] = {0, 0};
        int it = 0;
        for (int t = w; t < n_tiles; t += 2, it++) {
            const int pair0 = first + t * kPRows;
            /* columns from this one on see the token; all of the warp's see all, and are pairs, or not */
            const long long from = (long long)(j - before) * a.group - pair0;
            const int c0 = (int)max(0ll, min((long long)kPRows, from)), c1 = min(kPRows, pairs - pair0);
            const bool masked = __any_sync(0xffffffffu, c0 > 0) || c1 < kPRows;
            if (!at_warp_wait(&s_full[w], (uint32_t)it & 1u, abort_flag)) { give_up(); break; }
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < 4; c++) {
                uint32_t s[32];
                __syncwarp();
                at_ld32(tS + (uint32_t)(c * 32), s);
                const float4 *of = reinterpret_cast<const float4 *>(&pair_s[t % kWRing][c * 32]);
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    const float4 p = of[k / 2];
                    const float2 x = vb_f2_get(vb_f2_fma(vb_f2_pack(__uint_as_float(s[k]), __uint_as_float(s[k + 1])), vb_f2_mul(up2, vb_f2_pack(p.x, p.z)), vb_f2_pack(-p.y, -p.w)));
                    float e0 = exp2_fast(x.x), e1 = exp2_fast(x.y);
                    if (masked) {
                        if (c * 32 + k < c0 || c * 32 + k >= c1) e0 = 0.0f;
                        if (c * 32 + k + 1 < c0 || c * 32 + k + 1 >= c1) e1 = 0.0f;
                    }
                    sums[(k >> 1) & 1] = vb_f2_add(sums[(k >> 1) & 1], vb_f2_pack(e0, e1));
                }
            }
            tc_fence_before();
            vb_mbar_arrive(&s_empty[w]);
        }
        const float2 both = vb_f2_get(vb_f2_add(sums[0], sums[1]));
        const float sum = both.x + both.y;
        if (w == 1) sum_s[r] = sum;
        vb_named_bar(1, 256);
        if (w == 0 && j < span.length && !*(volatile int *)&far_s) {
            pdl_wait();
            const size_t at = ((size_t)seq * a.c.kv_heads + kv_head) * a.c.capacity + j;
            a.mass_out[at] = sum + sum_s[r] + (a.mass_in && j < before ? a.mass_in[at] : 0.0f);
        }
    } else if (warp < kWMmaWarp) {
        /* ---- queries: a warp has 16 pairs of a tile, NB * 8 lanes a pair, as in the attention ---- */
        constexpr int kLanes = NB * 8, kSide = 32 / kLanes, kBatch = 16 / kSide;
        const int lw = warp - 8, side = lane / kLanes, d = (lane - side * kLanes) * 4;
        const bool mine = side < kSide;
        pdl_wait();                                                        /* lse */
        for (int t = 0; t < n_tiles; t++) {
            const int slot = t % kWSlots, p0 = first + t * kPRows + lw * 16;
            ServeRaw4<T> raw[kBatch];
            float lse = 0.0f;
            /* a place on from pair to pair: a division for each took longer than the rest */
            int in_row = (p0 + side) / a.group;
            const T *p = q.data + seq * q.seq + in_row * q.row + kv_head * a.group * q.head + d;
            in_row = p0 + side - in_row * a.group;
            p += in_row * q.head;
#pragma unroll
            for (int u = 0; u < kBatch; u++) {
                const bool real = mine && p0 + u * kSide + side < pairs;
                raw[u].none();
                if (real) raw[u].load(p, a.wide);
                in_row += kSide;
                p += kSide * q.head;
                while (in_row >= a.group) {
                    in_row -= a.group;
                    p += q.row - a.group * q.head;
                }
            }
            if (lane < 16 && p0 + lane < pairs) {
                const int row = (p0 + lane) / a.group;
                lse = a.lse[((size_t)seq * a.max_rows + row) * a.heads + kv_head * a.group + p0 + lane - row * a.group];
            }
            if (!at_warp_wait(&q_empty[slot], ((uint32_t)(t / kWSlots) & 1u) ^ 1u, abort_flag)) { give_up(); break; }
            if (lane < 16) pair_s[t % kWRing][lw * 16 + lane].y = lse == -INFINITY ? INFINITY : lse * 1.44269504f;       /* a row without weights gives none */
#pragma unroll
            for (int u = 0; u < kBatch; u++) {
                const int r = lw * 16 + u * kSide + side;
                const float4 x = raw[u].get();
                uint32_t most = max(max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu), max(__float_as_uint(x.z) & 0x7fffffffu, __float_as_uint(x.w) & 0x7fffffffu));
                if constexpr (kSide == 1) {
                    most = __reduce_max_sync(0xffffffffu, most);
                } else {
#pragma unroll
                    for (int o = 1; o < kLanes; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
                }
                const uint32_t e = most >> 23, field = e == 0u || e == 255u ? 127u : min(268u - e, 253u);
                const float up = __uint_as_float(field << 23);
                if (!mine) continue;
                if (d == 0) pair_s[t % kWRing][r].x = a.scale * 1.44269504f * __uint_as_float((254u - field) << 23);
                unsigned char *to = q_s + slot * (QT * Cfg::kSlot) + (d >> 6) * kPBlock + at_off(r, (d & 63) >> 3) + (d & 7) * 2;
                const float y0 = x.x * up, y1 = x.y * up, y2 = x.z * up, y3 = x.w * up;
                const uint2 hi = make_uint2(half_pack(y0, y1), half_pack(y2, y3));
                *reinterpret_cast<uint2 *>(to) = hi;
                if constexpr (QT == 2) {
                    const float2 f = kv4_f2(hi.x), g = kv4_f2(hi.y);
                    *reinterpret_cast<uint2 *>(to + Cfg::kSlot) = make_uint2(half_pack(y0 - f.x, y1 - f.y), half_pack(y2 - g.x, y3 - g.y));
                }
            }
            at_proxy_fence();
            __syncwarp();
            if (lane == 0) vb_mbar_arrive(&q_full[slot]);
        }
    } else if (lane == 0) {
        /* ---- MMA issuer ---- */
        const uint32_t idesc = p_idesc(kPRows, false);
        const AtDesc k_desc(umma_desc_k_sw128(k_s)), q_desc(umma_desc_k_sw128(q_s));
        pdl_wait();
        bool ok = vb_mbar_wait(&k_full, 0u, abort_flag);
        for (int t = 0; t < n_tiles && ok; t++) {
            const int slot = t % kWSlots, w = t & 1;
            ok = vb_mbar_wait(&q_full[slot], (uint32_t)(t / kWSlots) & 1u, abort_flag) && vb_mbar_wait(&s_empty[w], ((uint32_t)(t >> 1) & 1u) ^ 1u, abort_flag);
            if (!ok) break;
            tc_fence_after();
            const AtDesc qd = q_desc.at(slot * (QT * Cfg::kSlot >> 4));
#pragma unroll
            for (int ks = 0; ks < NB * 2; ks++) {
                const int at = (ks >> 2) * (kPBlock >> 4) + 2 * (ks & 3);
#pragma unroll
                for (int u = 0; u < QT; u++) at_mma_ss(tmem + (uint32_t)(w * kPRows), k_desc.at(at), qd.at(at + u * (Cfg::kSlot >> 4)), idesc, ks + u != 0 ? 1u : 0u);
            }
            umma_commit(&q_empty[slot]);
            umma_commit(&s_full[w]);
        }
        if (!ok) give_up();
    }
    tc_fence_before();
    __syncthreads();
    if (*(volatile int *)&far_s) {
        /* scales too far apart: in fp32, a lane a token, four warps the pairs of 32 tokens in turn */
        pdl_wait();
        const Kv4Head head = kv4_head<NB>(a.c, a.c.row(seq, kv_head, 0));
        float *q_row = reinterpret_cast<float *>(base) + warp * NB * 32, *sums = reinterpret_cast<float *>(base) + 16 * NB * 32;
        const int j = tok0 + (warp & 3) * 32 + lane;
        if (warp < 16) {
            float sum = 0.0f;
            for (int p = first + (warp >> 2); p < pairs; p += 4) {
                const int row = p / a.group, h = kv_head * a.group + p - row * a.group;
                const float mul = kv4_plain_query<NB>(q.data + seq * q.seq + row * q.row + h * q.head, a.scale, q_row);
                const float lse = a.lse[((size_t)seq * a.max_rows + row) * a.heads + h], s = kv4_plain_score<NB>(head, min(j, span.length - 1), q_row, mul);
                if (j < before + row + 1 && lse != -INFINITY) sum += exp2_fast(s - lse * 1.44269504f);
                __syncwarp();
            }
            sums[warp * 32 + lane] = sum;
        }
        __syncthreads();
        if (warp < 4 && j < span.length) {
            const size_t at = ((size_t)seq * a.c.kv_heads + kv_head) * a.c.capacity + j;
            a.mass_out[at] = sums[warp * 32 + lane] + sums[(warp + 4) * 32 + lane] + sums[(warp + 8) * 32 + lane] + sums[(warp + 12) * 32 + lane] +
                             (a.mass_in && j < before ? a.mass_in[at] : 0.0f);
        }
    }
    if (warp == kWMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kWTmem) : "memory");
    }
}

template <int NB, class T>
int prompt_launch(Kv4Attn a, const ServeRows<T> &q, const ServeRows<T> &out, int sm_count, cudaStream_t st) {
    const long long row_tiles = ((long long)a.max_rows * a.group + kPRows - 1) / kPRows, units = row_tiles * a.c.kv_heads * a.c.seqs;
    if (units > INT_MAX) return serve_fail("too many rows");
    a.row_tiles = (int)row_tiles;
    a.split = units < sm_count && a.c.capacity > kPLeast * kPKeys;
    /* The units beyond the last whole round are cut where they are few and long: a part takes as long to begin and to end as five tiles, and
     * the join 4 us (512 units of eight tiles, 68 of them in the last round, cut in two: 130 us, not 110). */
    const int rest = (int)(units % sm_count), tiles = (a.c.capacity + kPKeys - 1) / kPKeys;
    a.tail_parts = !a.split && units > sm_count && rest > 0 && rest <= sm_count / 4 && tiles >= 16 ? std::min({sm_count / rest, kPTailParts, tiles / 4}) : 1;
    a.tail_units = a.tail_parts > 1 ? rest : 1;
    a.tail0 = a.tail_parts > 1 ? (int)units - rest : INT_MAX;
    const unsigned tail = a.tail_parts > 1 ? (unsigned)(rest * a.tail_parts) : 0u;
    const dim3 grid((unsigned)(a.split ? sm_count : tail ? units - rest + tail : units));
    const size_t smem = PCfg<NB, sizeof(T) == 4 ? 2 : 1>::kSmem;
    if (launch_pdl(kv4_prompt_kernel<NB, kWeightTerms<T>, T>, grid, dim3(kPThreads), smem, st, a, q, out) != cudaSuccess) return serve_launched() | -1;
    if ((a.split || tail) && launch_pdl(kv4_join_kernel<NB, T>, a.split ? grid : dim3(tail), dim3(kJThreads), 0, st, a, out) != cudaSuccess) return serve_launched() | -1;
    return 0;
}
template <int NB, class T>
int mass_many_launch(const Kv4Attn &a, const ServeRows<T> &q, cudaStream_t st) {
    const dim3 grid((unsigned)(((long long)a.c.capacity + kPKeys - 1) / kPKeys), a.c.kv_heads, a.c.seqs);
    const size_t smem = WCfg<NB, sizeof(T) == 4 ? 2 : 1>::kSmem;
    return launch_pdl(kv4_mass_many_kernel<NB, T>, grid, dim3(kWThreads), smem, st, a, q) == cudaSuccess ? 0 : serve_launched() | -1;
}
template <int NB, class T>
bool prompt_load() {
    cudaFuncAttributes f;
    if (cudaFuncGetAttributes(&f, kv4_join_kernel<NB, T>) != cudaSuccess) return false;
    if (cudaFuncSetAttribute(kv4_mass_many_kernel<NB, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, WCfg<NB, sizeof(T) == 4 ? 2 : 1>::kSmem) != cudaSuccess) return false;
    return cudaFuncSetAttribute(kv4_prompt_kernel<NB, kWeightTerms<T>, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, PCfg<NB, sizeof(T) == 4 ? 2 : 1>::kSmem) == cudaSuccess;
}

} // namespace

template <class T>
int kv4_prompt(const Kv4Attn &a, const ServeRows<T> &q, const ServeRows<T> &out, int sm_count, cudaStream_t st) {
    switch (a.c.blocks) {
    case 1: return prompt_launch<1, T>(a, q, out, sm_count, st);
    case 2: return prompt_launch<2, T>(a, q, out, sm_count, st);
    case 3: return prompt_launch<3, T>(a, q, out, sm_count, st);
    default: return prompt_launch<4, T>(a, q, out, sm_count, st);
    }
}
template <class T>
int kv4_mass_many(const Kv4Attn &a, const ServeRows<T> &q, cudaStream_t st) {
    switch (a.c.blocks) {
    case 1: return mass_many_launch<1, T>(a, q, st);
    case 2: return mass_many_launch<2, T>(a, q, st);
    case 3: return mass_many_launch<3, T>(a, q, st);
    default: return mass_many_launch<4, T>(a, q, st);
    }
}
template int kv4_mass_many<float>(const Kv4Attn &, const ServeRows<float> &, cudaStream_t);
template int kv4_mass_many<__nv_bfloat16>(const Kv4Attn &, const ServeRows<__nv_bfloat16> &, cudaStream_t);
template int kv4_mass_many<__half>(const Kv4Attn &, const ServeRows<__half> &, cudaStream_t);
template int kv4_prompt<float>(const Kv4Attn &, const ServeRows<float> &, const ServeRows<float> &, int, cudaStream_t);
template int kv4_prompt<__nv_bfloat16>(const Kv4Attn &, const ServeRows<__nv_bfloat16> &, const ServeRows<__nv_bfloat16> &, int, cudaStream_t);
template int kv4_prompt<__half>(const Kv4Attn &, const ServeRows<__half> &, const ServeRows<__half> &, int, cudaStream_t);

size_t kv4_prompt_floats(int blocks, int sm_count) { return blocks <= 4 ? (size_t)sm_count * kPRows * (blocks * 32 + 2) : 0; }
size_t kv4_aside_floats(int blocks, int sm_count) { return blocks <= 4 ? (size_t)sm_count * 2 * kPRows * blocks * 32 : 0; }

int kv4_prompt_load(int blocks) {
    bool ok = true;
    switch (blocks) {
    case 1: ok = prompt_load<1, float>() && prompt_load<1, __nv_bfloat16>() && prompt_load<1, __half>(); break;
    case 2: ok = prompt_load<2, float>() && prompt_load<2, __nv_bfloat16>() && prompt_load<2, __half>(); break;
    case 3: ok = prompt_load<3, float>() && prompt_load<3, __nv_bfloat16>() && prompt_load<3, __half>(); break;
    case 4: ok = prompt_load<4, float>() && prompt_load<4, __nv_bfloat16>() && prompt_load<4, __half>(); break;
    }
    return ok ? 0 : -1;
}

} // namespace vb

/*
 * vb_logprobs.cu - log probabilities of given tokens, entropy and the largest alternatives out of rows of logits, in one pass.
 *
 *   m = max x,  l = sum e^(x - m),  w = sum e^(x - m) (x - m);  lse = m + log l,  entropy = log l - w / l
 *
 * Bound by the logits' bytes where there are many rows (1024 fp32 rows of 100003: 80 us, 5.1 TB/s, 79 % of a plain copy's rate), by latency where
 * there is one (131072: 7.4 us). A row is split over the CTAs of a cluster;
 * a thread keeps m, l, w of what it reads, rescaled when its maximum rises. The largest values: a threshold that `top` values are known to reach (the
 * top-th largest of the maxima that 32 groups of threads have in their first stretch) lets a few dozen values of a row through, which are
 * collected and put in order at the end. Values are compared with their index below them, so all are different. Where more come through than
 * the list holds (rising rows), a CTA finds its largest again by bisection, from memory: slower and as right.
 */
#include <limits.h>
#include <type_traits>

#include "vb_serve.cuh"
#include "vb_tc.cuh"

namespace vb {

namespace {

constexpr int kLpThreads = 512, kLpWarps = kLpThreads / 32, kLpTop = 32, kLpList = 1024, kLpMaxSplit = 8;
/* vectors of 16 bytes that a thread takes at a time, with as many on their way: with four of BF16 it runs out of registers */
template <class T>
constexpr int kLpUnrolled = sizeof(T) == 4 ? 4 : 2;

struct LpArgs {
    const void *x;
    long long stride;
    int rows, vocab, top;
    const int *tokens;
    float *logprobs, *entropy;
    int *top_ids;
    float *top_logprobs;
};

/* Order of values as order of unsigned numbers: NaN above all, -0 as 0; the earlier index is the larger of two that tie. */
VB_DEVINL uint32_t lp_key(float v) {
    if (v != v) return 0xffffffffu;
    const uint32_t u = __float_as_uint(v + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
VB_DEVINL float lp_value(uint32_t key) {
    return key == 0xffffffffu ? __uint_as_float(0x7fffffffu) : __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
VB_DEVINL uint64_t lp_rank(float v, int i) { return ((uint64_t)lp_key(v) << 32) | (uint32_t)~i; }

struct LpSums {
    float m, l, w;
};
/* The same sums against a larger reference. Those of nothing stay nothing; one that vanishes takes its difference along: 0, not 0 * -inf */
VB_DEVINL void lp_rebase(LpSums &a, float m) {
    const float d = a.m - m, f = a.m > -INFINITY ? __expf(d) : 0.0f;
    a.w = f > 0.0f ? (a.w + a.l * d) * f : 0.0f;
    a.l *= f;
    a.m = m;
}
/* The sums of all lanes that differ in bits below N, in every lane */
template <int N>
VB_DEVINL void lp_join(LpSums &a) {
    float m = a.m;
#pragma unroll
    for (int o = 1; o < N; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    lp_rebase(a, m);
#pragma unroll
    for (int o = 1; o < N; o <<= 1) {
        a.l += __shfl_xor_sync(0xffffffffu, a.l, o);
        a.w += __shfl_xor_sync(0xffffffffu, a.w, o);
    }
}

/* The larger one; NaN where either is. */
VB_DEVINL float lp_max(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
VB_DEVINL float lp_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
/* 16 bytes of -inf: what stands in for vectors beyond a share */
template <class T>
constexpr uint32_t kLpNothing = std::is_same<T, float>::value ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;

template <class T>
VB_DEVINL void lp_values(const uint4 &r, float *v) {
    const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float2 f = serve_pair(u[j], (const T *)nullptr);
        if constexpr (sizeof(T) == 4) v[j] = f.x;
        else { v[2 * j] = f.x; v[2 * j + 1] = f.y; }
    }
}

/* How many of the `n` ranks in a list, largest first, are above v. */
VB_DEVINL int lp_above(const uint64_t *sorted, int n, uint64_t v) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sorted[mid] > v) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

template <class T>
__global__ void __launch_bounds__(kLpThreads, 2) logprobs_kernel(const LpArgs a) {
    constexpr int kEach = 16 / sizeof(T), kLpUnroll = kLpUnrolled<T>, kStep = kLpThreads * kLpUnroll;
    __shared__ uint64_t list[kLpList], best[kLpMaxSplit * kLpTop], group[32], threshold_s;
    __shared__ LpSums warp_sums[kLpWarps], cta_sums[kLpMaxSplit];
    __shared__ int n_list, bad_s[kLpMaxSplit], counts[kLpMaxSplit];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint32_t split, splits;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(split));
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(splits));
    /* waited for before anything is sent to another CTA's shared memory: by then that CTA runs */
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.x / splits;
    const T *x = static_cast<const T *>(a.x) + (long long)row * a.stride;
    /* elements before the first 16-byte boundary, then whole vectors, then the rest; this CTA's share of the vectors */
    const int head = min(a.vocab, (int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T)));
    const int vectors = (a.vocab - head) / kEach, tail = head + vectors * kEach;
    const int share = (vectors + splits - 1) / splits, v0 = min(vectors, (int)split * share), v1 = min(vectors, v0 + share);
    const uint4 *xv = reinterpret_cast<const uint4 *>(x + head);

    uint4 now[kLpUnroll], next[kLpUnroll];
    auto fetch = [&](int c0, uint4 (&r)[kLpUnroll]) {
#pragma unroll
        for (int u = 0; u < kLpUnroll; u++) {
            const int i = c0 + u * kLpThreads + tid;
            r[u] = i < v1 ? __ldcs(xv + i) : make_uint4(kLpNothing<T>, kLpNothing<T>, kLpNothing<T>, kLpNothing<T>);
        }
    };
    fetch(v0, now);
    /* the elements around the vectors go with the first CTA's first stretch, one a thread */
    float extra = -INFINITY, of_token = 0.0f;
    int extra_i = -1, token = -1;
    if (split == 0) {
        if (tid < head) extra_i = tid;
        else if (tid - head < a.vocab - tail) extra_i = tail + tid - head;
        if (extra_i >= 0) extra = serve_get(x + extra_i);
        if (tid == 0) {
            n_list = 0;
            if (a.tokens) token = a.tokens[row];
            if (token >= 0 && token < a.vocab) of_token = serve_get(x + token);
        }
    }
    if (tid == 0) { n_list = 0; threshold_s = 0; bad_s[0] = 0; }
    __syncthreads();

    LpSums sums = {-INFINITY, 0.0f, 0.0f};
    bool bad = false;                         /* NaN or +inf */
    /* the reference is the maximum: one that trailed by up to 8 left log probabilities near 0 differences of two numbers up to 8 */
    auto raise = [&](float top) {
        if (!(top <= sums.m)) {
            if (top < INFINITY) {
                lp_rebase(sums, top);
            } else {
                bad = true;
            }
        }
    };
    auto add = [&](float v) {
        const float d = fmaxf(v - sums.m, -150.0f), e = lp_ex2(d * 1.44269504f);      /* -inf: 0 and 0 * -150 */
        sums.l += e;
        sums.w = fmaf(e, d, sums.w);
    };
    uint64_t threshold = 0;
    float limit = -INFINITY;                  /* values from here on may be among the largest */
    auto collect = [&](float v, int i) {
        if (!(v < limit)) {
            const uint64_t r = lp_rank(v, i);
            if (r >= threshold) {
                const int at = atomicAdd(&n_list, 1);
                if (at < kLpList) list[at] = r;
            }
        }
    };
    for (int c0 = v0; c0 < v1 || c0 == v0; c0 += kStep) {
        const bool first = c0 == v0;
        if (c0 + kStep < v1) fetch(c0 + kStep, next);
        float top = first ? extra : -INFINITY, low = INFINITY;
#pragma unroll
        for (int u = 0; u < kLpUnroll; u++) {
            float v[kEach];
            lp_values<T>(now[u], v);
#pragma unroll
            for (int j = 0; j < kEach; j++) {
                top = lp_max(top, v[j]);
                low = fminf(low, v[j]);
            }
        }
        raise(top);
        if (first) add(extra);
        if (low - sums.m > -INFINITY) {
            /* two at a time; nothing is infinitely far below the reference, finite numbers more than fp32's largest apart neither */
            const uint64_t m2 = vb_f2_pack(-sums.m, -sums.m), log2e = vb_f2_pack(1.44269504f, 1.44269504f);
            uint64_t l2 = 0, w2 = 0;
#pragma unroll
            for (int u = 0; u < kLpUnroll; u++) {
                float v[kEach];
                lp_values<T>(now[u], v);
#pragma unroll
                for (int j = 0; j < kEach; j += 2) {
                    const uint64_t d = vb_f2_add(vb_f2_pack(v[j], v[j + 1]), m2);
                    const float2 x = vb_f2_get(vb_f2_mul(d, log2e));
                    const uint64_t e = vb_f2_pack(lp_ex2(x.x), lp_ex2(x.y));
                    l2 = vb_f2_add(l2, e);
                    w2 = vb_f2_fma(e, d, w2);
                }
            }
            const float2 l = vb_f2_get(l2), w = vb_f2_get(w2);
            sums.l += l.x + l.y;
            sums.w += w.x + w.y;
        } else {
#pragma unroll
            for (int u = 0; u < kLpUnroll; u++) {
                float v[kEach];
                lp_values<T>(now[u], v);
#pragma unroll
                for (int j = 0; j < kEach; j++) add(v[j]);
            }
        }
        if (a.top) {
            if (first) {
                /* this thread's largest, at its first place; those of 32 groups of threads; the top-th of them */
                int at = extra_i >= 0 && !(extra < top) ? extra_i : INT_MAX;      /* not below a NaN either: one that is none is put right */
#pragma unroll
                for (int u = 0; u < kLpUnroll; u++) {
                    const int i = c0 + u * kLpThreads + tid;
                    float v[kEach];
                    lp_values<T>(now[u], v);
                    if (i < v1)
#pragma unroll
                        for (int j = 0; j < kEach; j++)
                            if (top == top ? v[j] == top : v[j] != v[j]) at = min(at, head + i * kEach + j);
                }
                if (top != top && extra_i >= 0 && at == extra_i && extra == extra) at = INT_MAX;
                uint64_t most = at < INT_MAX ? lp_rank(top, at) : 0;
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
                if ((lane & 15) == 0) group[warp * 2 + (lane >> 4)] = most;
                __syncthreads();
                if (warp == 0) {
                    const uint64_t v = group[lane];
                    int rank = 0;
#pragma unroll
                    for (int o = 0; o < 32; o++) {
                        const uint64_t w = group[o];
                        rank += w > v || (w == v && o < lane);
                    }
                    if (rank == a.top - 1) threshold_s = v;
                }
                __syncthreads();
                threshold = threshold_s;
                limit = threshold == 0 ? -INFINITY : lp_value((uint32_t)(threshold >> 32));
                if (limit != limit) limit = INFINITY;      /* the threshold is a NaN: only NaN reaches it */
                if (extra_i >= 0) collect(extra, extra_i);
            }
            if (!(top < limit)) {
#pragma unroll
                for (int u = 0; u < kLpUnroll; u++) {
                    const int i = c0 + u * kLpThreads + tid;
                    float v[kEach];
                    lp_values<T>(now[u], v);
                    if (i < v1)
#pragma unroll
                        for (int j = 0; j < kEach; j++) collect(v[j], head + i * kEach + j);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kLpUnroll; u++) now[u] = next[u];
    }
    /* this CTA's sums: a warp's, then theirs */
    lp_join<32>(sums);
    if (lane == 0) warp_sums[warp] = sums;
    if (__any_sync(0xffffffffu, bad) && lane == 0) atomicOr(&bad_s[0], 1);
    __syncthreads();
    if (warp == kLpWarps - 1) {               /* the first warps have the list */
        sums = warp_sums[lane % kLpWarps];
        lp_join<kLpWarps>(sums);
        if (lane == 0) cta_sums[0] = sums;
    }
    /* this CTA's largest values, in order */
    const int there = min(a.top, (v1 - v0) * kEach + (split == 0 ? head + a.vocab - tail : 0));
    if (a.top) {
        int n = n_list;
        if (n > kLpList) {
            /* the largest rank that `there` of this CTA's values reach, a bit at a time; then those values alone */
            auto each = [&](auto &&f) {
                for (int i = v0 * kEach + tid; i < v1 * kEach; i += kLpThreads) f(serve_get(x + head + i), head + i);
                if (extra_i >= 0) f(extra, extra_i);
            };
            uint64_t least = 0;
            for (int bit = 63; bit >= 0; bit--) {
                const uint64_t trial = least | (1ull << bit);
                int reach = 0;
                each([&](float v, int i) { reach += lp_rank(v, i) >= trial; });
                __syncthreads();
                if (tid == 0) n_list = 0;
                __syncthreads();
                if (reach) atomicAdd(&n_list, reach);
                __syncthreads();
                if (n_list >= there) least = trial;
            }
            __syncthreads();
            if (tid == 0) n_list = 0;
            __syncthreads();
            threshold = least;
            limit = -INFINITY;
            each(collect);
            __syncthreads();
            n = n_list;
        }
        /* four threads count for a value */
        for (int i = tid >> 2; i < (n + 7) / 8 * 8; i += kLpThreads / 4) {
            const uint64_t v = i < n ? list[i] : 0;
            int rank = 0;
#pragma unroll 4
            for (int o = tid & 3; o < n; o += 4) rank += list[o] > v;
            rank += __shfl_xor_sync(0xffffffffu, rank, 1);
            rank += __shfl_xor_sync(0xffffffffu, rank, 2);
            if ((tid & 3) == 0 && i < n && rank < there) best[rank] = v;
        }
    }
    __syncthreads();
    /* to the cluster's first CTA */
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (splits > 1) {
        if (split != 0) {
            uint32_t to;
            if (tid < there) {
                asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(vb_smem_u32(&best[split * kLpTop + tid])));
                asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(best[tid]) : "memory");
            }
            if (tid == 0) {
                asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(vb_smem_u32(&cta_sums[split])));
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(cta_sums[0].m) : "memory");
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4), "f"(cta_sums[0].l) : "memory");
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 8), "f"(cta_sums[0].w) : "memory");
                asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(vb_smem_u32(&bad_s[split])));
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(bad_s[0]) : "memory");
                asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(vb_smem_u32(&counts[split])));
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(there) : "memory");
            }
        }
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (split != 0) return;
    }
    if (tid == 0) counts[0] = there;
    /* the row's sums, by every warp for itself */
    const bool in = lane < (int)splits;
    sums = in ? cta_sums[lane] : LpSums{-INFINITY, 0.0f, 0.0f};
    lp_join<kLpMaxSplit>(sums);
    sums.m = __shfl_sync(0xffffffffu, sums.m, 0);
    sums.l = __shfl_sync(0xffffffffu, sums.l, 0);
    const bool wrong = __any_sync(0xffffffffu, in && bad_s[in ? lane : 0] != 0);
    const float nan = __uint_as_float(0x7fffffffu), log_l = wrong ? nan : logf(sums.l);      /* -inf for a row of nothing but -inf */
    if (tid == 0) {
        if (a.logprobs) a.logprobs[row] = wrong || token < 0 || token >= a.vocab ? nan : sums.l == 0.0f ? -INFINITY : (of_token - sums.m) - log_l;
        if (a.entropy) a.entropy[row] = wrong ? nan : sums.l == 0.0f ? 0.0f : log_l - sums.w / sums.l;
    }
    if (!a.top) return;
    __syncthreads();                          /* counts[0] */
    /* a lane a value and a list (of eight, there or not): how many of the list are above the value */
    for (int i = tid >> 3; i < ((int)splits * a.top + 3) / 4 * 4; i += kLpThreads / 8) {
        const int c = i % (int)splits, k = i / (int)splits, o = tid & 7;
        const bool there_is = k < a.top && k < counts[c];
        const uint64_t v = there_is ? best[c * kLpTop + k] : 0;
        int rank = !there_is || o >= (int)splits ? 0 : o == c ? k : lp_above(best + o * kLpTop, counts[o], v);
#pragma unroll
        for (int x = 1; x < 8; x <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, x);
        if (!there_is || o != 0 || rank >= a.top) continue;
        const float value = lp_value((uint32_t)(v >> 32));
        const size_t to = (size_t)row * a.top + rank;
        if (a.top_ids) a.top_ids[to] = (int)~(uint32_t)v;
        if (a.top_logprobs) a.top_logprobs[to] = value == -INFINITY && log_l == log_l ? -INFINITY : (value - sums.m) - log_l;
    }
}

template <class T>
int logprobs_launch(const LpArgs &a, int sm_count, cudaStream_t st) {
    /* a row over more CTAs while there are SMs for them, each with a stretch of its own at least */
    constexpr int kStretch = kLpThreads * kLpUnrolled<T> * (16 / (int)sizeof(T));
    int splits = 1;
    while (splits < kLpMaxSplit && (long long)a.rows * splits * 2 <= 2 * sm_count && a.vocab >= splits * kStretch) splits *= 2;
    const cudaError_t e = launch_pdl_cluster(logprobs_kernel<T>, splits, dim3((unsigned)a.rows * splits), dim3(kLpThreads), 0, st, a);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return serve_fail(cudaGetErrorString(e));
    }
    return 0;
}

} // namespace

} // namespace vb

using namespace vb;

extern "C" int vb200_token_logprobs(const vb200_logprobs_t *a, void *stream) {
    if (!a || (!a->logits && a->rows > 0)) return serve_fail("no logits");
    if (a->type < VB200_F32 || a->type > VB200_F16) return serve_fail("logits are fp32, bf16 or fp16");
    if ((uintptr_t)a->logits % serve_size(a->type)) return serve_fail("logits have to be aligned to their elements");
    if (a->rows < 0 || a->rows > (1 << 27) || a->vocab < 1 || a->vocab > (1 << 30)) return serve_fail("rows have to be 0 to 2^27, vocab 1 to 2^30");
    if (a->top < 0 || a->top > kLpTop || a->top > a->vocab) return serve_fail("top has to be 0 to 32 and at most vocab");
    if (a->logprobs && !a->tokens) return serve_fail("logprobs needs tokens");
    if (a->rows == 0) return 0;
    int dev = 0, n_sm = 0, major = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess || major != 10) {
        cudaGetLastError();
        return serve_fail("an sm_100 GPU is required (there is no CPU fallback)");
    }
    if (!serve_on_device(a->logits)) return serve_fail("logits do not lie on the current device");
    if (serve_check({{a->tokens, "tokens"}, {a->logprobs, "logprobs"}, {a->entropy, "entropy"}, {a->top_ids, "top_ids"}, {a->top_logprobs, "top_logprobs"}})) return -1;
    const bool tops = a->top_ids || a->top_logprobs;
    const LpArgs l = {a->logits, a->row_stride, a->rows, a->vocab, tops ? a->top : 0, a->tokens, a->logprobs, a->entropy, a->top_ids, a->top_logprobs};
    const cudaStream_t st = (cudaStream_t)stream;
    if (a->type == VB200_F32) return logprobs_launch<float>(l, n_sm, st);
    if (a->type == VB200_BF16) return logprobs_launch<__nv_bfloat16>(l, n_sm, st);
    return logprobs_launch<__half>(l, n_sm, st);
}

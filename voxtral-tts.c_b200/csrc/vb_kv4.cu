/*
 * vb_kv4.cu - the key/value cache in 4 bits: its memory, rows into it and out of it, and eviction from it by
 * accumulated attention weight. Attention over it is in vb_kv4_attn.cu.
 */
#include <algorithm>
#include <limits.h>
#include <new>
#include <string>

#include "vb_kv4.cuh"
#include "vb_tc.cuh"

namespace vb {

namespace {
thread_local std::string g_serve_error;
}

int serve_fail(const char *what) {
    try {
        g_serve_error = what;
    } catch (...) {
    }
    return -1;
}
int serve_launched() {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : serve_fail(cudaGetErrorString(e));
}
bool serve_on_device(const void *p) {
    int now = 0;
    cudaPointerAttributes at;
    if (cudaGetDevice(&now) != cudaSuccess || cudaPointerGetAttributes(&at, p) != cudaSuccess) {
        cudaGetLastError();
        return false;
    }
    return at.type == cudaMemoryTypeManaged || (at.type == cudaMemoryTypeDevice && at.device == now);
}

namespace {

constexpr int kRowThreads = 256, kRowUnroll = 4;

/* ------------------------------------------------------------------ rows into the cache and out of it
 * A thread has words of 8 values: four lanes make a block of 32. The words of a token (keys, then values) lie side by side in the order of
 * threads; a CTA takes 1024 of them at a time, four a thread with their loads together. Memory-bound, and at one row a launch bound by its
 * latency. */
template <class T>
struct RowsArgs {
    Kv4 c;
    const int *lengths, *rows;
    int max_rows, wide;
    unsigned tokens;                                     /* seqs * max_rows */
    ServeRows<T> k, v;
};

template <int NB, class T, bool READ>
__global__ void __launch_bounds__(kRowThreads) kv4_rows_kernel(const RowsArgs<T> a) {
    constexpr unsigned kWords = NB * 4;                  /* of a row of a head */
    constexpr long long kChunk = kRowThreads * kRowUnroll;
    const unsigned plane = a.c.kv_heads * kWords, token_words = 2 * plane;
    const long long total = (long long)a.tokens * token_words;
    const int tid = threadIdx.x;
    pdl_launch_dependents();
    pdl_wait();
    for (long long c0 = blockIdx.x * kChunk; c0 < total; c0 += gridDim.x * kChunk) {
        const unsigned token0 = (unsigned)(c0 / token_words), off0 = (unsigned)(c0 - (long long)token0 * token_words);
        float v[kRowUnroll][8];
        uint32_t code[kRowUnroll], byte[kRowUnroll], w[kRowUnroll];
        size_t row[kRowUnroll];
        T *p[kRowUnroll];
        bool real[kRowUnroll], is_v[kRowUnroll];
#pragma unroll
        for (int u = 0; u < kRowUnroll; u++) {
            const unsigned o = off0 + u * kRowThreads + tid, ahead = o / token_words, rest = o - ahead * token_words;
            is_v[u] = rest >= plane;
            const unsigned in_plane = is_v[u] ? rest - plane : rest, h = in_plane / kWords;
            w[u] = in_plane - h * kWords;
            const bool in = token0 + ahead < a.tokens;
            const unsigned token = in ? token0 + ahead : 0, s = token / a.max_rows, r = token - s * a.max_rows;
            const Kv4Span span = kv4_span(a.lengths, a.rows, a.max_rows, s, a.c.capacity);
            const int slot = span.length - span.rows + (int)r;
            real[u] = in && (int)r < span.rows && slot >= 0;
            const ServeRows<T> &x = is_v[u] ? a.v : a.k;
            p[u] = x.data + (long long)s * x.seq + (long long)r * x.row + (long long)h * x.head + w[u] * 8;
            row[u] = a.c.row(s, h, real[u] ? slot : 0);
            if (!READ) {
#pragma unroll
                for (int j = 0; j < 8; j++) v[u][j] = 0.0f;
                if (real[u]) serve_load<8>(p[u], a.wide, v[u]);
            } else if (real[u]) {
                const uint8_t *base = (is_v[u] ? a.c.v : a.c.k) + row[u] * (NB * 16);
                if (!is_v[u]) {
                    code[u] = reinterpret_cast<const uint32_t *>(base)[kv4_key_word(w[u], NB)];
                } else if (kv4_whole(NB)) {
                    code[u] = reinterpret_cast<const uint32_t *>(base)[w[u]];
                } else {
                    const uint16_t *from = reinterpret_cast<const uint16_t *>(base);
                    code[u] = from[kv4_value_half(2 * w[u], NB)] | ((uint32_t)from[kv4_value_half(2 * w[u] + 1, NB)] << 16);
                }
                byte[u] = (is_v[u] ? a.c.vs : a.c.ks)[row[u] * NB + (w[u] >> 2)];
            }
        }
#pragma unroll
        for (int u = 0; u < kRowUnroll; u++) {
            if (!READ) {
                /* the largest magnitude by its bits, so that a NaN is the largest of all */
                uint32_t most = 0;
#pragma unroll
                for (int j = 0; j < 8; j++) most = max(most, __float_as_uint(v[u][j]) & 0x7fffffffu);
                most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
                if (!real[u]) continue;
                const uint32_t scale = kv4_scale(__uint_as_float(most));
                const uint32_t c = scale == 255u ? 0u : kv4_codes(v[u], kv4_inverse(scale));       /* a block that is NaN: codes of zero */
                uint8_t *base = (is_v[u] ? a.c.v : a.c.k) + row[u] * (NB * 16);
                if (!is_v[u]) {
                    reinterpret_cast<uint32_t *>(base)[kv4_key_word(w[u], NB)] = c;
                } else if (kv4_whole(NB)) {
                    reinterpret_cast<uint32_t *>(base)[w[u]] = c;
                } else {
                    uint16_t *to = reinterpret_cast<uint16_t *>(base);
                    to[kv4_value_half(2 * w[u], NB)] = (uint16_t)c;
                    to[kv4_value_half(2 * w[u] + 1, NB)] = (uint16_t)(c >> 16);
                }
                if ((w[u] & 3) == 0) (is_v[u] ? a.c.vs : a.c.ks)[row[u] * NB + (w[u] >> 2)] = (uint8_t)scale;
            } else {
                if (!real[u]) code[u] = byte[u] = 0;
                const float scale = kv4_scale_value(byte[u]);
                uint32_t half[4];
                kv4_halves(code[u], half);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float2 f = kv4_f2(half[j]);
                    v[u][2 * j] = f.x * scale;
                    v[u][2 * j + 1] = f.y * scale;
                }
                if constexpr (sizeof(T) == 4) {
                    /* two lanes' 64 bytes, 32 of them a store: whole sectors (the words of a pair are one token's and one head's) */
                    const bool odd = tid & 1;
                    float other[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float give = odd ? v[u][j] : v[u][4 + j];
                        other[j] = __shfl_xor_sync(0xffffffffu, give, 1);
                    }
                    if (!real[u]) continue;
                    if (a.wide) {
                        float4 *to = reinterpret_cast<float4 *>(p[u] - (odd ? 8 : 0)) + (odd ? 1 : 0);
                        to[0] = odd ? make_float4(other[0], other[1], other[2], other[3]) : make_float4(v[u][0], v[u][1], v[u][2], v[u][3]);
                        to[2] = odd ? make_float4(v[u][4], v[u][5], v[u][6], v[u][7]) : make_float4(other[0], other[1], other[2], other[3]);
                        continue;
                    }
                }
                if (real[u]) serve_store<8>(p[u], a.wide, v[u]);
            }
        }
    }
}

template <int NB, class T>
int rows_launch(const vb200_kv4 *h, const vb200_kv4_rows_t &a, bool read, cudaStream_t st) {
    RowsArgs<T> r = {h->c, a.lengths, a.rows, a.max_rows, 0, (unsigned)h->c.seqs * a.max_rows, serve_rows<T>(a.k), serve_rows<T>(a.v)};
    r.wide = serve_wide(r.k) && serve_wide(r.v);
    const long long words = (long long)r.tokens * h->c.kv_heads * NB * 8, chunk = kRowThreads * kRowUnroll;
    const unsigned grid = (unsigned)std::min((words + chunk - 1) / chunk, (long long)h->w.sm_count * 16);
    const cudaError_t e = launch_pdl(read ? kv4_rows_kernel<NB, T, true> : kv4_rows_kernel<NB, T, false>, dim3(grid), dim3(kRowThreads), 0, st, r);
    return e == cudaSuccess ? 0 : serve_launched() | -1;
}

template <class T>
int rows_dims(const vb200_kv4 *h, const vb200_kv4_rows_t &a, bool read, cudaStream_t st) {
#define VB_CALL(n) rows_launch<n, T>(h, a, read, st)
    VB_KV4_DIMS(h->c.blocks, VB_CALL)
#undef VB_CALL
}

/* ------------------------------------------------------------------ eviction */
struct EvictArgs {
    Kv4 from, into;
    const int *lengths;
    int *new_lengths;
    const float *mass;
    float *new_mass;
    long long new_mass_ld;
    int *kept;
    int keep, recent, first, in_place;
};

/* Order of masses as order of unsigned numbers; NaN below all, -0 as 0. */
VB_DEVINL uint32_t evict_key(float m) {
    if (m != m) return 0u;
    const uint32_t u = __float_as_uint(m + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelThreads = 1024, kSelEach = 32, kSelChunk = kSelThreads * kSelEach, kSelBins = 2048;

/* Which tokens stay: a CTA per sequence and head. The need-th largest key of the middle by digits of 11, 11 and 10 bits (counts of a
 * digit among those that share the digits before it; the first holds sign, exponent and two bits, so that masses spread over it), then
 * the tokens in order. A thread keeps the keys of up to 32 tokens in registers; longer sequences are read again, 32768 tokens at a time.
 */
__global__ void __launch_bounds__(kSelThreads) kv4_select_kernel(const EvictArgs a) {
    __shared__ int count[kSelBins], warp_sum[32];
    __shared__ uint2 place[kSelEach * 32];                /* of a warp's 32 tokens: how many stay, how many tie; then how many before them */
    __shared__ uint2 warp_place[32];
    __shared__ uint32_t prefix;
    __shared__ int want;
    const int s = blockIdx.y, h = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_launch_dependents();
    pdl_wait();
    const int n = min(max(a.lengths[s], 0), a.from.capacity);
    int *kept = a.kept + ((size_t)s * a.from.kv_heads + h) * a.keep;
    if (n <= a.keep) {
        for (int i = tid; i < n; i += kSelThreads) kept[i] = i;
        return;
    }
    const float *mass = a.mass + ((size_t)s * a.from.kv_heads + h) * a.from.capacity;
    const int lo = a.first, hi = n - a.recent;            /* the middle; it holds more than are needed of it */
    uint32_t key[kSelEach];
    auto read = [&](int c0) {
#pragma unroll
        for (int j = 0; j < kSelEach; j++) {
            const int i = c0 + j * kSelThreads + tid;
            if (i < n) key[j] = evict_key(mass[i]);
            if (c0 + (j + 1) * kSelThreads >= n) break;
        }
    };
    const bool once = n <= kSelChunk;
    if (once) read(0);
    if (tid == 0) { prefix = 0; want = a.keep - a.first - a.recent; }
    const bool none = a.keep == a.first + a.recent;
    if (!none) {
        int shift = 21;
#pragma unroll 1
        for (int pass = 0; pass < 3; pass++) {
            const uint32_t mask = pass == 0 ? 0u : pass == 1 ? 0xffe00000u : 0xfffffc00u, digit = pass == 2 ? 1023u : 2047u;
            for (int x = tid; x < kSelBins; x += kSelThreads) count[x] = 0;
            __syncthreads();
            const uint32_t p = prefix;
            for (int c0 = 0; c0 < n; c0 += kSelChunk) {
                if (!once) read(c0);
#pragma unroll
                for (int j = 0; j < kSelEach; j++) {
                    const int i = c0 + j * kSelThreads + tid;
                    if (i >= lo && i < hi && (key[j] & mask) == p) atomicAdd(&count[(key[j] >> shift) & digit], 1);
                    if (c0 + (j + 1) * kSelThreads >= n) break;
                }
            }
            __syncthreads();
            /* thread x has bins 2047 - 2 x and 2046 - 2 x: how many lie above them */
            const int left = want, b1 = kSelBins - 1 - 2 * tid, n1 = count[b1], n0 = count[b1 - 1];
            int above = n1 + n0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, above, o);
                if (lane >= o) above += v;
            }
            if (lane == 31) warp_sum[warp] = above;
            __syncthreads();
            if (warp == 0) {
                int v = warp_sum[lane];
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int u = __shfl_up_sync(0xffffffffu, v, o);
                    if (lane >= o) v += u;
                }
                warp_sum[lane] = v;
            }
            __syncthreads();
            above += (warp ? warp_sum[warp - 1] : 0) - n1 - n0;
            if (above < left && left <= above + n1) { prefix = p | ((uint32_t)b1 << shift); want = left - above; }
            else if (above + n1 < left && left <= above + n1 + n0) { prefix = p | ((uint32_t)(b1 - 1) << shift); want = left - above - n1; }
            __syncthreads();
            shift = pass == 0 ? 10 : 0;
        }
    }
    __syncthreads();
    /* of those equal to the threshold the first `ties` stay */
    const uint32_t threshold = prefix;
    const int ties = want;
    uint2 base = make_uint2(0, 0);                        /* stay, tie, before this chunk */
    for (int c0 = 0; c0 < n; c0 += kSelChunk) {
        if (!once) read(c0);
        uint32_t stay = 0, tie = 0;                       /* a bit a token */
#pragma unroll
        for (int j = 0; j < kSelEach; j++) {
            const int i = c0 + j * kSelThreads + tid;
            const bool edge = i < lo || i >= hi;
            const bool is_sure = i < n && (edge || (!none && key[j] > threshold)), is_tie = i < n && !edge && !none && key[j] == threshold;
            const unsigned bs = __ballot_sync(0xffffffffu, is_sure), bt = __ballot_sync(0xffffffffu, is_tie);
            stay |= (uint32_t)is_sure << j;
            tie |= (uint32_t)is_tie << j;
            if (lane == 0) place[j * 32 + warp] = make_uint2(__popc(bs), __popc(bt));
        }
        __syncthreads();
        {
            uint2 v = place[tid];
            const uint2 own = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned x = __shfl_up_sync(0xffffffffu, v.x, o), y = __shfl_up_sync(0xffffffffu, v.y, o);
                if (lane >= o) { v.x += x; v.y += y; }
            }
            if (lane == 31) warp_place[warp] = v;
            __syncthreads();
            if (warp == 0) {
                uint2 t = warp_place[lane];
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned x = __shfl_up_sync(0xffffffffu, t.x, o), y = __shfl_up_sync(0xffffffffu, t.y, o);
                    if (lane >= o) { t.x += x; t.y += y; }
                }
                warp_place[lane] = t;
            }
            __syncthreads();
            const uint2 ahead = warp ? warp_place[warp - 1] : make_uint2(0, 0);
            place[tid] = make_uint2(base.x + ahead.x + v.x - own.x, base.y + ahead.y + v.y - own.y);
            base.x += warp_place[31].x;
            base.y += warp_place[31].y;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kSelEach; j++) {
            if (c0 + j * kSelThreads >= n) break;
            const bool is_sure = (stay >> j) & 1u, is_tie = (tie >> j) & 1u;
            const unsigned bs = __ballot_sync(0xffffffffu, is_sure), bt = __ballot_sync(0xffffffffu, is_tie), below = (1u << lane) - 1u;
            const uint2 at = place[j * 32 + warp];
            const int tied = (int)at.y + __popc(bt & below);
            if (is_sure || (is_tie && tied < ties)) kept[(int)at.x + __popc(bs & below) + min(tied, ties)] = c0 + j * kSelThreads + tid;
        }
        __syncthreads();
    }
}

/* The rows that stay into their places, in pieces of 16 bytes (codes) and a byte a block (scales). In place a CTA takes all of a
 * head, since a row's new slot may be another row's old one: rows move towards the front in order, so a stretch may be written once all
 * stretches up to it have been read. */
constexpr int kMoveThreads = 256;

template <bool IN_PLACE>
__global__ void __launch_bounds__(kMoveThreads) kv4_move_kernel(const EvictArgs a) {
    const int s = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
    pdl_launch_dependents();
    pdl_wait();
    const int n = min(max(a.lengths[s], 0), a.from.capacity), m = min(n, a.keep);
    if (blockIdx.x == 0 && h == 0 && tid == 0) a.new_lengths[s] = m;     /* whoever reads it later finds the same m */
    const int blocks = a.from.blocks, pieces = blocks;                   /* of 16 bytes a row and plane */
    const int per = kMoveThreads / (2 * pieces);                         /* rows at a time */
    const int r0 = tid / (2 * pieces), piece = tid - r0 * 2 * pieces;
    const bool is_v = piece >= pieces;
    const int *kept = a.kept + ((size_t)s * a.from.kv_heads + h) * a.keep;
    const size_t from0 = a.from.row(s, h, 0), into0 = a.into.row(s, h, 0), head = (size_t)s * a.from.kv_heads + h;
    const int first = IN_PLACE ? 0 : blockIdx.x * per, step = IN_PLACE ? per : gridDim.x * per;
    if (IN_PLACE && m == n && (!a.new_mass || a.new_mass == a.mass)) return;      /* nothing moves */
    for (int i0 = first; i0 < m; i0 += step) {
        const int i = i0 + r0;
        const bool mine = r0 < per && i < m;
        uint4 v = make_uint4(0, 0, 0, 0);
        uint8_t scale = 0;
        float mass = 0.0f;
        const int col = is_v ? piece - pieces : piece;
        if (mine) {
            const size_t row = from0 + kept[i];
            v = reinterpret_cast<const uint4 *>(is_v ? a.from.v : a.from.k)[row * pieces + col];
            scale = (is_v ? a.from.vs : a.from.ks)[row * blocks + col];
            if (piece == 0 && a.new_mass) mass = a.mass[head * a.from.capacity + kept[i]];
        }
        if (IN_PLACE) __syncthreads();
        if (mine) {
            const size_t row = into0 + i;
            reinterpret_cast<uint4 *>(is_v ? a.into.v : a.into.k)[row * pieces + col] = v;
            (is_v ? a.into.vs : a.into.ks)[row * blocks + col] = scale;
            if (piece == 0 && a.new_mass) a.new_mass[head * a.new_mass_ld + i] = mass;
        }
    }
}

/* Loads the kernels on the current device: nothing is left to be loaded inside a capture. */
template <int NB>
int rows_load() {
    cudaFuncAttributes f;
    const void *kernels[] = {(const void *)kv4_rows_kernel<NB, float, false>, (const void *)kv4_rows_kernel<NB, float, true>,
                             (const void *)kv4_rows_kernel<NB, __nv_bfloat16, false>, (const void *)kv4_rows_kernel<NB, __nv_bfloat16, true>,
                             (const void *)kv4_rows_kernel<NB, __half, false>, (const void *)kv4_rows_kernel<NB, __half, true>,
                             (const void *)kv4_select_kernel, (const void *)kv4_move_kernel<false>, (const void *)kv4_move_kernel<true>};
    for (const void *k : kernels)
        if (cudaFuncGetAttributes(&f, k) != cudaSuccess) return serve_launched() | -1;
    return 0;
}
int load(int blocks) {
    if (kv4_attention_load(blocks)) return -1;
#define VB_CALL(n) rows_load<n>()
    VB_KV4_DIMS(blocks, VB_CALL)
#undef VB_CALL
}

int check_rows(const vb200_kv4 *h, const vb200_kv4_rows_t *a) {
    if (!h || !a) return serve_fail("no cache or no arguments");
    if (!a->lengths || !a->k.data || !a->v.data) return serve_fail("lengths, k and v are needed");
    if (a->max_rows < 0) return serve_fail("max_rows is negative");
    if (a->k.type != a->v.type || a->k.type < VB200_F32 || a->k.type > VB200_F16) return serve_fail("k and v are of one type: fp32, bf16 or fp16");
    if (((uintptr_t)a->k.data | (uintptr_t)a->v.data) % serve_size(a->k.type)) return serve_fail("k and v have to be aligned to their elements");
    int now = -1;
    if (cudaGetDevice(&now) != cudaSuccess || now != h->device) return serve_fail("the cache lies on another device than the current one");
    if (!serve_on_device(a->k.data)) return serve_fail("k does not lie on the current device");
    return 0;
}

int rows_call(const vb200_kv4 *h, const vb200_kv4_rows_t *a, bool read, cudaStream_t st) {
    if (check_rows(h, a)) return -1;
    if (a->max_rows == 0) return 0;
    if ((long long)a->max_rows * h->c.seqs > INT_MAX) return serve_fail("too many rows");
    if (a->k.type == VB200_F32) return rows_dims<float>(h, *a, read, st);
    if (a->k.type == VB200_BF16) return rows_dims<__nv_bfloat16>(h, *a, read, st);
    return rows_dims<__half>(h, *a, read, st);
}

} // namespace

} // namespace vb

using namespace vb;

extern "C" {

const char *vb200_serve_error(void) { return g_serve_error.c_str(); }

vb200_kv4_t *vb200_kv4_open(int seqs, int kv_heads, int head_dim, int capacity) {
    const bool dim_ok = head_dim == 32 || head_dim == 64 || head_dim == 96 || head_dim == 128 || head_dim == 192 || head_dim == 256;
    if (!dim_ok) { serve_fail("head_dim has to be 32, 64, 96, 128, 192 or 256"); return nullptr; }
    if (seqs < 1 || seqs > 65535 || kv_heads < 1 || kv_heads > 65535 || capacity < 1 || capacity > (1 << 30)) {
        serve_fail("seqs and kv_heads have to be 1 to 65535, capacity 1 to 2^30");
        return nullptr;
    }
    int dev = 0, major = 0, minor = 0, n_sm = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || major != 10 || minor != 0) {
        cudaGetLastError();
        serve_fail("an sm_100 GPU is required (there is no CPU fallback)");
        return nullptr;
    }
    vb200_kv4 *h = new (std::nothrow) vb200_kv4();
    if (!h) { serve_fail("out of memory"); return nullptr; }
    if (load(head_dim / 32)) {
        delete h;
        return nullptr;
    }
    h->device = dev;
    h->head_dim = head_dim;
    Kv4 &c = h->c;
    c.seqs = seqs; c.kv_heads = kv_heads; c.blocks = head_dim / 32; c.capacity = capacity;
    c.slots = (capacity + kKv4Tile - 1) / kKv4Tile * kKv4Tile;
    /* partial results of as many CTAs as run at once, 16 rows each */
    h->w.sm_count = n_sm;
    h->w.n_tickets = 4 * n_sm;
    h->w.part_floats = (size_t)4 * n_sm * 16 * (head_dim + 2);
    const size_t rows = (size_t)seqs * kv_heads * c.slots, codes = rows * (size_t)(head_dim / 2), scales = rows * (size_t)c.blocks;
    const size_t work = h->w.part_floats * sizeof(float), tickets = sizeof(unsigned) * (size_t)(h->w.n_tickets + 1);
    h->bytes = 2 * codes + 2 * scales + work + tickets;
    void *p = nullptr;
    if (cudaMalloc(&p, h->bytes) != cudaSuccess || cudaMemset(p, 0, h->bytes) != cudaSuccess || cudaDeviceSynchronize() != cudaSuccess) {
        cudaGetLastError();
        if (p) cudaFree(p);
        delete h;
        serve_fail("out of device memory for the cache");
        return nullptr;
    }
    h->base = p;
    c.k = (uint8_t *)p;                        /* every plane is a multiple of 64 bytes */
    c.v = c.k + codes;
    c.ks = c.v + codes;
    c.vs = c.ks + scales;
    h->w.part = (float *)(c.vs + scales);
    h->w.tickets = (unsigned *)(h->w.part + h->w.part_floats);
    h->w.status = (int *)(h->w.tickets + h->w.n_tickets);
    return h;
}

void vb200_kv4_close(vb200_kv4_t *h) {
    if (!h) return;
    int now = -1;
    if (cudaGetDevice(&now) == cudaSuccess && now != h->device) cudaSetDevice(h->device);
    cudaFree(h->base);
    if (now >= 0 && now != h->device) cudaSetDevice(now);
    delete h;
}

int vb200_kv4_status(const vb200_kv4_t *h) {
    if (!h) return serve_fail("no cache");
    int s = 0;
    if (cudaMemcpy(&s, h->w.status, sizeof(int), cudaMemcpyDeviceToHost) != cudaSuccess) return serve_launched() ? -1 : serve_fail("the status could not be read");
    return s;
}

size_t vb200_kv4_bytes(const vb200_kv4_t *h) { return h ? h->bytes : 0; }

int vb200_kv4_append(vb200_kv4_t *h, const vb200_kv4_rows_t *a, void *stream) { return rows_call(h, a, false, (cudaStream_t)stream); }
int vb200_kv4_read(const vb200_kv4_t *h, const vb200_kv4_rows_t *a, void *stream) { return rows_call(h, a, true, (cudaStream_t)stream); }

int vb200_kv4_evict(vb200_kv4_t *h, vb200_kv4_t *into, const vb200_kv4_evict_t *a, void *stream) {
    if (!h || !into || !a) return serve_fail("no cache or no arguments");
    if (!a->lengths || !a->new_lengths || !a->mass || !a->kept) return serve_fail("lengths, new_lengths, mass and kept are needed");
    if (a->keep < 1 || a->recent < 0 || a->first < 0 || (long long)a->recent + a->first > a->keep)
        return serve_fail("keep has to be positive, recent and first not negative and together at most keep");
    if (into->c.seqs != h->c.seqs || into->c.kv_heads != h->c.kv_heads || into->c.blocks != h->c.blocks) return serve_fail("into has other seqs, kv_heads or head_dim");
    if (a->keep > into->c.capacity) return serve_fail("keep is more than into holds");
    if (a->new_mass && a->new_mass_ld < a->keep) return serve_fail("new_mass_ld is less than keep");
    if (a->new_mass == a->mass && (into != h || a->new_mass_ld != h->c.capacity)) return serve_fail("new_mass may be mass only where into is the cache itself and new_mass_ld its capacity");
    int now = -1;
    if (cudaGetDevice(&now) != cudaSuccess || now != h->device || into->device != h->device) return serve_fail("a cache lies on another device than the current one");
    if (!serve_on_device(a->mass)) return serve_fail("mass does not lie on the current device");
    const cudaStream_t st = (cudaStream_t)stream;
    EvictArgs e = {h->c, into->c, a->lengths, a->new_lengths, a->mass, a->new_mass, a->new_mass_ld, a->kept, a->keep, a->recent, a->first, into == h};
    cudaError_t err = launch_pdl(kv4_select_kernel, dim3(h->c.kv_heads, h->c.seqs), dim3(kSelThreads), 0, st, e);
    if (err != cudaSuccess) return serve_launched() | -1;
    if (into == h) {
        err = launch_pdl(kv4_move_kernel<true>, dim3(1, h->c.kv_heads, h->c.seqs), dim3(kMoveThreads), 0, st, e);
    } else {
        const int per = kMoveThreads / (2 * h->c.blocks);
        const long long chunks = ((long long)a->keep + per - 1) / per, heads = (long long)h->c.kv_heads * h->c.seqs;
        const long long most = std::max(1ll, (long long)h->w.sm_count * 16 / heads);
        err = launch_pdl(kv4_move_kernel<false>, dim3((unsigned)std::min(chunks, most), h->c.kv_heads, h->c.seqs), dim3(kMoveThreads), 0, st, e);
    }
    return err == cudaSuccess ? 0 : serve_launched() | -1;
}

int vb200_kv4_attention(vb200_kv4_t *h, const vb200_kv4_attention_t *a, void *stream) {
    if (!h || !a) return serve_fail("no cache or no arguments");
    if (!a->lengths || !a->q.data || !a->out.data) return serve_fail("lengths, q and out are needed");
    if (a->max_rows < 0) return serve_fail("max_rows is negative");
    if (a->heads < 1 || a->heads % h->c.kv_heads) return serve_fail("heads has to be a multiple of the cache's kv_heads");
    if (a->q.type != a->out.type || a->q.type < VB200_F32 || a->q.type > VB200_F16) return serve_fail("q and out are of one type: fp32, bf16 or fp16");
    if (((uintptr_t)a->q.data | (uintptr_t)a->out.data) % serve_size(a->q.type)) return serve_fail("q and out have to be aligned to their elements");
    if (a->mass_in && !a->mass_out) return serve_fail("mass_in without mass_out");
    if (a->mass_out && !a->lse) return serve_fail("mass_out needs lse");
    if (!(a->scale > -1e30f && a->scale < 1e30f)) return serve_fail("scale is not a finite number");
    int now = -1;
    if (cudaGetDevice(&now) != cudaSuccess || now != h->device) return serve_fail("the cache lies on another device than the current one");
    if (!serve_on_device(a->q.data)) return serve_fail("q does not lie on the current device");
    if (a->max_rows == 0 && !a->mass_out) return 0;
    return kv4_attention(h->c, h->w, *a, (cudaStream_t)stream);
}

} /* extern "C" */

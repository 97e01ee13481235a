/*
 * vb_kv4.cu - the key/value cache in 4 bits: its memory, rows into it and out of it, and eviction from it by
 * accumulated attention weight. Attention over it is in vb_kv4_attn.cu.
 */
#include <algorithm>
#include <limits.h>
#include <stdio.h>
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
int serve_check(std::initializer_list<ServePointer> pointers) {
    int now = -1;
    cudaGetDevice(&now);
    for (const ServePointer &x : pointers) {
        if (!x.p) continue;
        cudaPointerAttributes at;
        if (cudaPointerGetAttributes(&at, x.p) != cudaSuccess) {
            cudaGetLastError();
            at.type = cudaMemoryTypeUnregistered;
        }
        if ((at.type == cudaMemoryTypeDevice && at.device == now) || at.type == cudaMemoryTypeManaged || (at.type == cudaMemoryTypeHost && at.devicePointer == x.p)) continue;
        char what[96];
        snprintf(what, sizeof what, "%s does not lie on the current device", x.name);
        return serve_fail(what);
    }
    return 0;
}

namespace {

constexpr int kRowThreads = 256, kRowUnroll = 4;

/* ------------------------------------------------------------------ rows into the cache and out of it
 * A CTA has rows of one head, keys or values; a thread a word of 8 values of a row, four rows at a time with their loads together; four
 * lanes make a block of 32. Memory-bound, and at one row a launch bound by its latency: 4097 bf16 rows of two sequences and 8 heads of 128
 * in and out again as fp32, 118 MB, 24 us, 4.8 TB/s; one row of eight sequences in and out 6.5 us, the host's time for two launches. (With
 * words of all heads side by side, indices worked out word by word, 4097 rows of two sequences took 22 us in and 16 out.) */
template <class T>
struct RowsArgs {
    Kv4 c;
    const int *lengths, *rows;
    int max_rows, wide;
    ServeRows<T> k, v;
};

template <int NB, class T, bool READ>
__global__ void __launch_bounds__(kRowThreads) kv4_rows_kernel(const RowsArgs<T> a) {
    constexpr int kWords = NB * 4;                                       /* of a row */
    const int kRows = (int)blockDim.x / kWords;                          /* rows side by side */
    const int tid = threadIdx.x, w = tid % kWords, r0 = tid / kWords, h = blockIdx.y >> 1, s = blockIdx.z;
    const bool is_v = blockIdx.y & 1;
    pdl_launch_dependents();
    pdl_wait();
    const Kv4Span span = kv4_span(a.lengths, a.rows, a.max_rows, s, a.c.capacity);
    const int before = span.length - span.rows;                          /* slot of row 0 */
    T *x = (is_v ? a.v.data + s * a.v.seq + h * a.v.head : a.k.data + s * a.k.seq + h * a.k.head) + w * 8;
    const long long ld = is_v ? a.v.row : a.k.row;
    const size_t row0 = a.c.row(s, h, 0);
    uint8_t *codes = (is_v ? a.c.v : a.c.k) + row0 * (NB * 16), *scales = (is_v ? a.c.vs : a.c.ks) + row0 * NB + (w >> 2);
    /* where this thread's word lies in a row of codes; values of 96 and 192 as two half words */
    const int at = is_v ? kv4_value_half(2 * w, NB) * 2 : kv4_key_word(w, NB) * 4, at2 = kv4_value_half(2 * w + 1, NB) * 2;
    const bool halves = !kv4_whole(NB) && is_v;
    for (int c0 = blockIdx.x * (kRows * kRowUnroll); c0 < span.rows; c0 += gridDim.x * (kRows * kRowUnroll)) {
        float v[kRowUnroll][8];
        uint32_t code[kRowUnroll], byte[kRowUnroll];
        bool real[kRowUnroll];
#pragma unroll
        for (int u = 0; u < kRowUnroll; u++) {
            const int r = c0 + u * kRows + r0, slot = before + r;
            real[u] = r0 < kRows && r < span.rows && slot >= 0;
            if (!READ) {
#pragma unroll
                for (int j = 0; j < 8; j++) v[u][j] = 0.0f;
                if (real[u]) serve_load<8>(x + r * ld, a.wide, v[u]);
            } else {
                code[u] = byte[u] = 0;
                if (real[u]) {
                    const uint8_t *base = codes + (size_t)slot * (NB * 16);
                    code[u] = halves ? *reinterpret_cast<const uint16_t *>(base + at) | ((uint32_t) * reinterpret_cast<const uint16_t *>(base + at2) << 16)
                                     : *reinterpret_cast<const uint32_t *>(base + at);
                    byte[u] = scales[(size_t)slot * NB];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kRowUnroll; u++) {
            const int r = c0 + u * kRows + r0;
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
                uint8_t *base = codes + (size_t)(before + r) * (NB * 16);
                if (halves) {
                    *reinterpret_cast<uint16_t *>(base + at) = (uint16_t)c;
                    *reinterpret_cast<uint16_t *>(base + at2) = (uint16_t)(c >> 16);
                } else {
                    *reinterpret_cast<uint32_t *>(base + at) = c;
                }
                if ((w & 3) == 0) scales[(size_t)(before + r) * NB] = (uint8_t)scale;
            } else {
                const float scale = kv4_scale_value(byte[u]);
                uint32_t half[4];
                kv4_halves(code[u], half);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float2 f = kv4_f2(half[j]);
                    v[u][2 * j] = f.x * scale;
                    v[u][2 * j + 1] = f.y * scale;
                }
                T *p = x + r * ld;
                if constexpr (sizeof(T) == 4) {
                    /* two lanes' 64 bytes, 32 of them a store: whole sectors (the words of a pair are one row's) */
                    const bool odd = tid & 1;
                    float other[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float give = odd ? v[u][j] : v[u][4 + j];
                        other[j] = __shfl_xor_sync(0xffffffffu, give, 1);
                    }
                    if (!real[u]) continue;
                    if (a.wide) {
                        float4 *to = reinterpret_cast<float4 *>(p - (odd ? 8 : 0)) + (odd ? 1 : 0);
                        to[0] = odd ? make_float4(other[0], other[1], other[2], other[3]) : make_float4(v[u][0], v[u][1], v[u][2], v[u][3]);
                        to[2] = odd ? make_float4(v[u][4], v[u][5], v[u][6], v[u][7]) : make_float4(other[0], other[1], other[2], other[3]);
                        continue;
                    }
                }
                if (real[u]) serve_store<8>(p, a.wide, v[u]);
            }
        }
    }
}

template <int NB, class T>
int rows_launch(const vb200_kv4 *h, const vb200_kv4_rows_t &a, bool read, cudaStream_t st) {
    RowsArgs<T> r = {h->c, a.lengths, a.rows, a.max_rows, 0, serve_rows<T>(a.k), serve_rows<T>(a.v)};
    r.wide = serve_wide(r.k) && serve_wide(r.v);
    /* a row or two are a warp or two: CTAs of full size take 0.9 us longer to be there */
    const int threads = (int)std::min<long long>(kRowThreads, ((long long)a.max_rows * NB * 4 + 31) / 32 * 32), kEach = threads / (NB * 4) * kRowUnroll;
    const long long heads = 2ll * h->c.kv_heads * h->c.seqs, chunks = (a.max_rows + kEach - 1) / kEach;
    const long long most = std::max(1ll, (long long)h->w.sm_count * 64 / heads);
    const dim3 grid((unsigned)std::min(chunks, most), 2 * h->c.kv_heads, h->c.seqs);
    const cudaError_t e = launch_pdl(read ? kv4_rows_kernel<NB, T, true> : kv4_rows_kernel<NB, T, false>, grid, dim3(threads), 0, st, r);
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

constexpr int kSelThreads = 1024, kSelBins = 2048, kSelHeld = 40960;

/* Which tokens stay: a CTA per sequence and head. The need-th largest key of the middle by digits of 11, 11 and 10 bits (counts of a
 * digit among those that share the digits before it; the first holds sign, exponent and two bits, so that masses spread over it), then
 * the tokens in order: a thread has a stretch of them, an odd number so that threads' reads fall on different banks. Keys wait in shared
 * memory; of sequences too long for that they are read again. Bound by the latencies of its passes: 26 us for 128 heads of 32768 tokens. (With a thread's 32 keys in registers, loops unrolled over them:
 * 17 us for 1601 tokens and 44 for 32768, most of it for fetching the code.) */
__global__ void __launch_bounds__(kSelThreads) kv4_select_kernel(const EvictArgs a) {
    extern __shared__ uint32_t held[];
    __shared__ int count[kSelBins], warp_sum[32];
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
    const bool hold = n <= kSelHeld;
    auto key_of = [&](int i) { return hold ? held[i] : evict_key(mass[i]); };
    if (hold) {
#pragma unroll 8
        for (int i = tid; i < n; i += kSelThreads) held[i] = evict_key(mass[i]);
    }
    for (int x = tid; x < kSelBins; x += kSelThreads) count[x] = 0;
    if (tid == 0) { prefix = 0; want = a.keep - a.first - a.recent; }
    __syncthreads();
    const bool none = a.keep == a.first + a.recent;
    if (!none) {
#pragma unroll 1
        for (int pass = 0; pass < 3; pass++) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
            const uint32_t mask = pass == 0 ? 0u : pass == 1 ? 0xffe00000u : 0xfffffc00u, digit = pass == 2 ? 1023u : 2047u, p = prefix;
#pragma unroll 4
            for (int i = lo + tid; i < hi; i += kSelThreads) {
                const uint32_t key = key_of(i);
                if ((key & mask) == p) atomicAdd(&count[(key >> shift) & digit], 1);
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
            count[b1] = count[b1 - 1] = 0;                /* for the next pass */
            __syncthreads();
            int ahead = warp_sum[lane];
            ahead = lane < warp ? ahead : 0;
            above += (int)__reduce_add_sync(0xffffffffu, (unsigned)ahead) - n1 - n0;
            if (above < left && left <= above + n1) { prefix = p | ((uint32_t)b1 << shift); want = left - above; }
            else if (above + n1 < left && left <= above + n1 + n0) { prefix = p | ((uint32_t)(b1 - 1) << shift); want = left - above - n1; }
            __syncthreads();
        }
    }
    /* of those equal to the threshold the first `ties` stay */
    const uint32_t threshold = prefix;
    const int ties = want, each = ((n + kSelThreads - 1) / kSelThreads) | 1, i0 = min(n, tid * each), i1 = min(n, i0 + each);
    uint2 here = make_uint2(0, 0);                        /* of this thread's tokens: how many stay, how many tie */
    for (int i = i0; i < i1; i++) {
        const uint32_t key = key_of(i);
        const bool edge = i < lo || i >= hi;
        here.x += edge || (!none && key > threshold);
        here.y += !edge && !none && key == threshold;
    }
    uint2 upto = here;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned x = __shfl_up_sync(0xffffffffu, upto.x, o), y = __shfl_up_sync(0xffffffffu, upto.y, o);
        if (lane >= o) { upto.x += x; upto.y += y; }
    }
    if (lane == 31) warp_place[warp] = upto;
    __syncthreads();
    const uint2 t = lane < warp ? warp_place[lane] : make_uint2(0, 0);
    int stay = (int)(upto.x - here.x + __reduce_add_sync(0xffffffffu, t.x)), tied = (int)(upto.y - here.y + __reduce_add_sync(0xffffffffu, t.y));
    for (int i = i0; i < i1; i++) {
        const uint32_t key = key_of(i);
        const bool edge = i < lo || i >= hi, is_tie = !edge && !none && key == threshold;
        const bool stays = edge || (!none && key > threshold) || (is_tie && tied < ties);
        if (stays) kept[stay + min(tied, ties)] = i;
        stay += stays && !is_tie;
        tied += is_tie;
    }
}
size_t select_smem(int capacity) { return sizeof(uint32_t) * (size_t)std::min(capacity, kSelHeld); }

/* The rows that stay into their places, in pieces of 16 bytes (codes) and a byte a block (scales). In place a CTA takes all of a
 * head, since a row's new slot may be another row's old one: rows move towards the front in order, so a stretch may be written once all
 * stretches up to it have been read. 128 heads of 8192 rows of 128 dims out of 32768: 62 us, 4.6 TB/s read and written. */
constexpr int kMoveThreads = 256;

template <bool IN_PLACE>
__global__ void __launch_bounds__(kMoveThreads) kv4_move_kernel(const EvictArgs a) {
    const int s = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
    pdl_launch_dependents();
    pdl_wait();
    const int n = min(max(a.lengths[s], 0), a.from.capacity), m = min(n, a.keep);
    if (blockIdx.x == 0 && h == 0 && tid == 0) a.new_lengths[s] = m;     /* may be lengths: whoever reads it later finds another n but the same m */
    const int blocks = a.from.blocks, pieces = blocks;                   /* of 16 bytes a row and plane */
    const int per = kMoveThreads / (2 * pieces);                         /* rows at a time */
    const int r0 = tid / (2 * pieces), piece = tid - r0 * 2 * pieces;
    const bool is_v = piece >= pieces;
    const int *kept = a.kept + ((size_t)s * a.from.kv_heads + h) * a.keep;
    const size_t from0 = a.from.row(s, h, 0), into0 = a.into.row(s, h, 0), head = (size_t)s * a.from.kv_heads + h;
    const int first = IN_PLACE ? 0 : blockIdx.x * per, step = IN_PLACE ? per : gridDim.x * per;
    /* nothing moves: tokens stay in order, so where the last one is at its place all are */
    if (IN_PLACE && (m == 0 || kept[m - 1] == m - 1) && (!a.new_mass || a.new_mass == a.mass)) return;
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
    if (cudaFuncSetAttribute(kv4_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)select_smem(kSelHeld)) != cudaSuccess) return serve_launched() | -1;
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
    if (a->max_rows < 0) return serve_fail("max_rows is negative");
    if (!a->lengths || (a->max_rows > 0 && (!a->k.data || !a->v.data))) return serve_fail("lengths, k and v are needed");
    if (a->k.type != a->v.type || a->k.type < VB200_F32 || a->k.type > VB200_F16) return serve_fail("k and v are of one type: fp32, bf16 or fp16");
    if (((uintptr_t)a->k.data | (uintptr_t)a->v.data) % serve_size(a->k.type)) return serve_fail("k and v have to be aligned to their elements");
    int now = -1;
    if (cudaGetDevice(&now) != cudaSuccess || now != h->device) return serve_fail("the cache lies on another device than the current one");
    if (a->max_rows == 0) return 0;
    if (!serve_on_device(a->k.data)) return serve_fail("k does not lie on the current device");
    return serve_check({{a->v.data, "v"}, {a->lengths, "lengths"}, {a->rows, "rows"}});
}

int rows_call(const vb200_kv4 *h, const vb200_kv4_rows_t *a, bool read, cudaStream_t st) {
    if (check_rows(h, a)) return -1;
    if (a->max_rows == 0) return 0;
    if (a->max_rows > (1 << 30)) return serve_fail("max_rows is more than 2^30");
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
    if (seqs < 1 || seqs > 65535 || kv_heads < 1 || kv_heads > 16384 || capacity < 1 || capacity > (1 << 30)) {
        serve_fail("seqs have to be 1 to 65535, kv_heads 1 to 16384, capacity 1 to 2^30");
        return nullptr;
    }
    /* in 128 bits: sizes within these limits can pass 64 */
    if ((unsigned __int128)seqs * kv_heads * ((capacity + kKv4Tile - 1) / kKv4Tile * kKv4Tile) * (head_dim + head_dim / 16) > (unsigned __int128)1 << 40) {
        serve_fail("seqs, kv_heads, capacity and head_dim have to be less: rows of more than 2^40 bytes");
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
    /* partial results of as many CTAs as run at once: two an SM of eight rows, or one of 128 */
    h->w.sm_count = n_sm;
    h->w.n_tickets = 2 * n_sm;
    h->w.part_floats = std::max((size_t)2 * n_sm * 8 * (head_dim + 2), kv4_prompt_floats(head_dim / 32, n_sm));
    const size_t rows = (size_t)seqs * kv_heads * c.slots, codes = rows * (size_t)(head_dim / 2), scales = rows * (size_t)c.blocks;
    const size_t aside = kv4_aside_floats(c.blocks, n_sm), work = (h->w.part_floats + aside) * sizeof(float), tickets = sizeof(unsigned) * (size_t)(h->w.n_tickets + n_sm + 1);
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
    h->w.aside = h->w.part + h->w.part_floats;
    h->w.tickets = (unsigned *)(h->w.aside + aside);
    h->w.rooms = h->w.tickets + h->w.n_tickets;
    h->w.status = (int *)(h->w.rooms + n_sm);
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
    int s = 0, now = -1;
    if (cudaGetDevice(&now) == cudaSuccess && now != h->device) cudaSetDevice(h->device);
    /* streams that do not wait for the default one have to be waited for by themselves */
    bool read = cudaDeviceSynchronize() == cudaSuccess && cudaMemcpy(&s, h->w.status, sizeof(int), cudaMemcpyDeviceToHost) == cudaSuccess;
    /* said once: what is queued from here on begins anew (tickets and rooms are given back where a wait runs out too) */
    if (read && s) read = cudaMemset(h->w.status, 0, sizeof(int)) == cudaSuccess && cudaDeviceSynchronize() == cudaSuccess;
    if (!read && !serve_launched()) serve_fail("the status could not be read");
    if (now >= 0 && now != h->device) cudaSetDevice(now);
    return read ? s : -1;
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
    if (serve_check({{a->lengths, "lengths"}, {a->new_lengths, "new_lengths"}, {a->new_mass, "new_mass"}, {a->kept, "kept"}})) return -1;
    const cudaStream_t st = (cudaStream_t)stream;
    EvictArgs e = {h->c, into->c, a->lengths, a->new_lengths, a->mass, a->new_mass, a->new_mass_ld, a->kept, a->keep, a->recent, a->first, into == h};
    cudaError_t err = launch_pdl(kv4_select_kernel, dim3(h->c.kv_heads, h->c.seqs), dim3(kSelThreads), select_smem(h->c.capacity), st, e);
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
    if (a->max_rows < 0) return serve_fail("max_rows is negative");
    if (!a->lengths || (a->max_rows > 0 && (!a->q.data || !a->out.data))) return serve_fail("lengths, q and out are needed");
    if (a->heads < 1 || a->heads % h->c.kv_heads) return serve_fail("heads has to be a multiple of the cache's kv_heads");
    if (a->q.type != a->out.type || a->q.type < VB200_F32 || a->q.type > VB200_F16) return serve_fail("q and out are of one type: fp32, bf16 or fp16");
    if (((uintptr_t)a->q.data | (uintptr_t)a->out.data) % serve_size(a->q.type)) return serve_fail("q and out have to be aligned to their elements");
    if (a->mass_in && !a->mass_out) return serve_fail("mass_in without mass_out");
    if (a->mass_out && a->max_rows > 0 && !a->lse) return serve_fail("mass_out needs lse");
    if (!(a->scale > -1e30f && a->scale < 1e30f)) return serve_fail("scale is not a finite number");
    int now = -1;
    if (cudaGetDevice(&now) != cudaSuccess || now != h->device) return serve_fail("the cache lies on another device than the current one");
    if (a->max_rows > 0 && !serve_on_device(a->q.data)) return serve_fail("q does not lie on the current device");
    if (a->max_rows == 0 && !a->mass_out) return 0;
    if (a->max_rows > 0 && serve_check({{a->out.data, "out"}, {a->lse, "lse"}})) return -1;
    if (serve_check({{a->lengths, "lengths"}, {a->rows, "rows"}, {a->mass_in, "mass_in"}, {a->mass_out, "mass_out"}})) return -1;
    return kv4_attention(h->c, h->w, *a, (cudaStream_t)stream);
}

} /* extern "C" */

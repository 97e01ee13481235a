/*
 * vb_kv4.cu - the key/value cache in 4 bits: its memory, rows into it and out of it, and eviction from it by
 * accumulated attention weight. Attention over it is in vb_kv4_attn.cu.
 */
#include <algorithm>
#include <new>
#include <string>

#include "vb_serve.cuh"

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

constexpr int kRowThreads = 256;

/* ------------------------------------------------------------------ rows into the cache and out of it
 * A thread has a word (8 values): four lanes make a block of 32. Both planes in one launch: blockIdx.y. Memory-bound, and at one row a
 * launch bound by its latency. */
template <class T>
struct RowsArgs {
    Kv4 c;
    const int *lengths, *rows;
    int max_rows, wide;
    ServeRows<T> k, v;
};

template <class T, bool READ>
__global__ void __launch_bounds__(kRowThreads) kv4_rows_kernel(const RowsArgs<T> a) {
    const int words = a.c.blocks * 4;                    /* of a row of a head */
    const long long total = (long long)a.c.seqs * a.max_rows * a.c.kv_heads * words;
    const bool is_v = blockIdx.y != 0;
    const ServeRows<T> &x = is_v ? a.v : a.k;
    uint8_t *codes = is_v ? a.c.v : a.c.k, *scales = is_v ? a.c.vs : a.c.ks;
    /* whole warps stay together: the four lanes of a block share its scale */
    for (long long i0 = ((long long)blockIdx.x * kRowThreads + threadIdx.x) & ~31ll; i0 < total; i0 += (long long)gridDim.x * kRowThreads) {
        const long long i = i0 + (threadIdx.x & 31);
        const bool in = i < total;
        const long long at = in ? i : total - 1;
        const int w = (int)(at % words);
        const long long rest = at / words;
        const int h = (int)(rest % a.c.kv_heads);
        const long long sr = rest / a.c.kv_heads;
        const int r = (int)(sr % a.max_rows), s = (int)(sr / a.max_rows);
        const Kv4Span span = kv4_span(a.lengths, a.rows, a.max_rows, s, a.c.capacity);
        const int slot = span.length - span.rows + r;
        const bool real = in && r < span.rows && slot >= 0;
        T *p = x.data + s * x.seq + r * x.row + h * x.head + w * 8;
        const size_t row = a.c.row(s, h, real ? slot : 0);
        uint8_t *base = codes + row * (size_t)(a.c.blocks * 16);
        float v[8];
        if (!READ) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = 0.0f;
            if (real) serve_load<8>(p, a.wide, v);
            /* the largest magnitude by its bits, so that a NaN is the largest of all */
            uint32_t most = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            if (!real) continue;
            const uint32_t byte = kv4_scale(__uint_as_float(most));
            const uint32_t code = byte == 255u ? 0u : kv4_codes(v, kv4_inverse(byte));       /* a block that is NaN: codes of zero */
            if (is_v) {
                uint16_t *to = reinterpret_cast<uint16_t *>(base);
                to[kv4_value_half(2 * w, a.c.blocks)] = (uint16_t)code;
                to[kv4_value_half(2 * w + 1, a.c.blocks)] = (uint16_t)(code >> 16);
            } else {
                reinterpret_cast<uint32_t *>(base)[kv4_key_word(w, a.c.blocks)] = code;
            }
            if ((w & 3) == 0) scales[row * a.c.blocks + (w >> 2)] = (uint8_t)byte;
        } else {
            if (!real) continue;
            uint32_t code;
            if (is_v) {
                const uint16_t *from = reinterpret_cast<const uint16_t *>(base);
                code = from[kv4_value_half(2 * w, a.c.blocks)] | ((uint32_t)from[kv4_value_half(2 * w + 1, a.c.blocks)] << 16);
            } else {
                code = reinterpret_cast<const uint32_t *>(base)[kv4_key_word(w, a.c.blocks)];
            }
            const float scale = kv4_scale_value(scales[row * a.c.blocks + (w >> 2)]);
            uint32_t half[4];
            kv4_halves(code, half);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 f = kv4_f2(half[j]);
                v[2 * j] = f.x * scale;
                v[2 * j + 1] = f.y * scale;
            }
            serve_store<8>(p, a.wide, v);
        }
    }
}

template <class T>
int rows_launch(const vb200_kv4 *h, const vb200_kv4_rows_t &a, bool read, cudaStream_t st) {
    RowsArgs<T> r = {h->c, a.lengths, a.rows, a.max_rows, 0, serve_rows<T>(a.k), serve_rows<T>(a.v)};
    r.wide = serve_wide(r.k) && serve_wide(r.v);
    const long long words = (long long)h->c.seqs * a.max_rows * h->c.kv_heads * h->c.blocks * 4;
    const long long most = (long long)h->w.sm_count * 16;
    const dim3 grid((unsigned)std::min((words + kRowThreads - 1) / kRowThreads, most), 2);
    if (read) kv4_rows_kernel<T, true><<<grid, kRowThreads, 0, st>>>(r);
    else kv4_rows_kernel<T, false><<<grid, kRowThreads, 0, st>>>(r);
    return serve_launched();
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

constexpr int kSelThreads = 1024;

/* Which tokens stay: a CTA per sequence and head. The need-th largest key of the middle by four passes of 8 bits (counts of a
 * digit among those that share the digits before it), then the tokens in order. */
__global__ void __launch_bounds__(kSelThreads) kv4_select_kernel(const EvictArgs a) {
    __shared__ int count[256], warp_sum[32][2], base[2];
    __shared__ uint32_t prefix;
    __shared__ int want;
    const int s = blockIdx.y, h = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = min(max(a.lengths[s], 0), a.from.capacity);
    int *kept = a.kept + ((size_t)s * a.from.kv_heads + h) * a.keep;
    if (n <= a.keep) {
        for (int i = tid; i < n; i += kSelThreads) kept[i] = i;
        return;
    }
    const float *mass = a.mass + ((size_t)s * a.from.kv_heads + h) * a.from.capacity;
    const int lo = a.first, hi = n - a.recent;            /* the middle; it holds more than are needed of it */
    if (tid == 0) { prefix = 0; want = a.keep - a.first - a.recent; }
    if (a.keep > a.first + a.recent) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) count[tid] = 0;
            __syncthreads();
            const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8), p = prefix;
            for (int i = lo + tid; i < hi; i += kSelThreads) {
                const uint32_t key = evict_key(mass[i]);
                if ((key & mask) == p) atomicAdd(&count[(key >> shift) & 255u], 1);
            }
            __syncthreads();
            if (tid == 0) {
                int left = want, d = 255;
                for (; d > 0 && count[d] < left; d--) left -= count[d];
                prefix = p | ((uint32_t)d << shift);
                want = left;
            }
            __syncthreads();
        }
    }
    __syncthreads();
    /* of those equal to the threshold the first `ties` stay */
    const bool none = a.keep == a.first + a.recent;
    const uint32_t threshold = prefix;
    const int ties = want;
    if (tid == 0) base[0] = base[1] = 0;
    __syncthreads();
    for (int i0 = 0; i0 < n; i0 += kSelThreads) {
        const int i = i0 + tid;
        bool sure = false, tie = false;
        if (i < n) {
            if (i < lo || i >= hi) sure = true;
            else if (!none) {
                const uint32_t key = evict_key(mass[i]);
                sure = key > threshold;
                tie = key == threshold;
            }
        }
        const unsigned bt = __ballot_sync(0xffffffffu, tie), bs = __ballot_sync(0xffffffffu, sure);
        if (lane == 0) { warp_sum[warp][0] = __popc(bs); warp_sum[warp][1] = __popc(bt); }
        __syncthreads();
        int sures = base[0], tied = base[1];
        for (int w = 0; w < warp; w++) { sures += warp_sum[w][0]; tied += warp_sum[w][1]; }
        const unsigned below = (1u << lane) - 1u;
        const int my_ties = tied + __popc(bt & below);
        if (sure || (tie && my_ties < ties)) kept[sures + __popc(bs & below) + min(my_ties, ties)] = i;
        __syncthreads();
        if (tid == kSelThreads - 1) { base[0] = sures + __popc(bs); base[1] = tied + __popc(bt); }
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
int rows_load() {
    cudaFuncAttributes f;
    const void *kernels[] = {(const void *)kv4_rows_kernel<float, false>, (const void *)kv4_rows_kernel<float, true>,
                             (const void *)kv4_rows_kernel<__nv_bfloat16, false>, (const void *)kv4_rows_kernel<__nv_bfloat16, true>,
                             (const void *)kv4_rows_kernel<__half, false>, (const void *)kv4_rows_kernel<__half, true>,
                             (const void *)kv4_select_kernel, (const void *)kv4_move_kernel<false>, (const void *)kv4_move_kernel<true>};
    for (const void *k : kernels)
        if (cudaFuncGetAttributes(&f, k) != cudaSuccess) return serve_launched() | -1;
    return 0;
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
    if (a->k.type == VB200_F32) return rows_launch<float>(h, *a, read, st);
    if (a->k.type == VB200_BF16) return rows_launch<__nv_bfloat16>(h, *a, read, st);
    return rows_launch<__half>(h, *a, read, st);
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
    if (rows_load() || kv4_attention_load(head_dim / 32)) {
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
    kv4_select_kernel<<<dim3(h->c.kv_heads, h->c.seqs), kSelThreads, 0, st>>>(e);
    if (serve_launched()) return -1;
    if (into == h) {
        kv4_move_kernel<true><<<dim3(1, h->c.kv_heads, h->c.seqs), kMoveThreads, 0, st>>>(e);
    } else {
        const int per = kMoveThreads / (2 * h->c.blocks);
        const long long chunks = ((long long)a->keep + per - 1) / per, heads = (long long)h->c.kv_heads * h->c.seqs;
        const long long most = std::max(1ll, (long long)h->w.sm_count * 16 / heads);
        kv4_move_kernel<false><<<dim3((unsigned)std::min(chunks, most), h->c.kv_heads, h->c.seqs), kMoveThreads, 0, st>>>(e);
    }
    return serve_launched();
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

/*
 * vb_serve.cuh - what the operators of voxtral_b200_serve.h share: the cache's layout in device memory and
 * its 4-bit format, element types, the host side's errors.
 */
#ifndef VB_SERVE_CUH
#define VB_SERVE_CUH

#include <cuda_fp16.h>

#include <initializer_list>

#include "../../include/voxtral_b200_serve.h"
#include "vb_common.cuh"

namespace vb {

/* ------------------------------------------------------------------ host */
/* Says why a call failed; returns -1. */
int serve_fail(const char *what);
int serve_launched();                                     /* 0, or -1 with the launch's error */
/* Whether `p` lies on the current device (or is managed memory). */
bool serve_on_device(const void *p);
/* 0 where all of them are NULL or memory that a kernel of the current device may use (host memory that is mapped, too); -1 with the name of the
 * first that is not. What a kernel does with other pointers is a fault of the GPU's. */
struct ServePointer {
    const void *p;
    const char *name;
};
int serve_check(std::initializer_list<ServePointer> pointers);

template <class T>
struct ServeRows {                                        /* vb200_rows_t with its type */
    T *data;
    long long seq, row, head;
};
template <class T>
ServeRows<T> serve_rows(const vb200_rows_t &r) { return {static_cast<T *>(r.data), r.seq, r.row, r.head}; }
inline size_t serve_size(int type) { return type == VB200_F32 ? 4 : 2; }

/* ------------------------------------------------------------------ the cache's layout
 * [seq][kv head][slot] rows, keys and values, codes and scale bytes each in a plane of their own. Slots are padded to whole
 * tiles of 64, so that a tile of them can be read whatever the length.
 *
 * Inside a row, the codes are ordered for the lanes of a warp-level MMA (m16n8k16: lane = 4 g + t) so that what a lane
 * takes from a row lies side by side:
 *   keys    lane t takes 8 values (a word) of every block of 32: word (t, block) holds values 32 block + 8 t ..
 *   values  lane g takes head_dim / 8 values: those from g * head_dim / 8 on where that stays within a block (1, 2, 4, 8 blocks), else
 *           4 of every block: half word (g, block) holds values 32 block + 4 g ..
 * Two values a byte, the earlier one in the low half. */
constexpr int kKv4Tile = 64;

struct Kv4 {
    uint8_t *k, *v, *ks, *vs;
    int seqs, kv_heads, blocks, capacity, slots;          /* blocks of 32 a row; slots: capacity in whole tiles */
    VB_DEVINL size_t row(int seq, int head, int slot) const { return ((size_t)seq * kv_heads + head) * slots + slot; }
};

__host__ __device__ constexpr bool kv4_whole(int blocks) { return (blocks & (blocks - 1)) == 0; }
/* Where natural word w (values 8 w ..) of a key row lies; where natural half word u (values 4 u ..) of a value row does. */
VB_DEVINL int kv4_key_word(int w, int blocks) { return (w & 3) * blocks + (w >> 2); }
VB_DEVINL int kv4_value_half(int u, int blocks) { return kv4_whole(blocks) ? u : (u & 7) * blocks + (u >> 3); }

/* lengths and rows as the calls read them */
struct Kv4Span {
    int length, rows;
};
VB_DEVINL Kv4Span kv4_span(const int *lengths, const int *rows, int max_rows, int seq, int capacity) {
    Kv4Span s;
    s.length = min(max(lengths[seq], 0), capacity);
    s.rows = rows ? min(max(rows[seq], 0), max_rows) : max_rows;
    return s;
}

/* ------------------------------------------------------------------ the format */
/* Scale byte of a block: `most` its largest magnitude, infinite or NaN where a value is. Subnormal numbers have the byte of 2^-126, a block of
 * zeros 0: it is not far below any other. */
VB_DEVINL uint32_t kv4_scale(float most) {
    const uint32_t e = __float_as_uint(most) >> 23;
    return e == 255u ? 255u : most == 0.0f ? 0u : e <= 3u ? 1u : e - 2u;
}
/* A block with this byte is not exact in FP16 based on the scale byte `top`: its least value, half a scale, lies below FP16's smallest step
 * where `top` stands for 2^13. */
constexpr int kKv4Range = 36;
VB_DEVINL bool kv4_far(uint32_t byte, int top) { return byte != 0u && byte != 255u && (int)byte + kKv4Range < top; }
/* 1 / scale, for bytes 1 .. 252: exact (0: any finite number does) */
VB_DEVINL float kv4_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
/* Eight values times `inv` as codes (byte i: values 2 i, 2 i + 1). */
VB_DEVINL uint32_t kv4_codes(const float (&x)[8], float inv) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(x[0] * inv), "f"(x[1] * inv), "f"(x[2] * inv), "f"(x[3] * inv), "f"(x[4] * inv), "f"(x[5] * inv), "f"(x[6] * inv), "f"(x[7] * inv));
    return r;
}
/* The four bytes of a word as pairs of FP16 numbers, the low code's in the low half: exact. */
VB_DEVINL void kv4_halves(uint32_t w, uint32_t (&r)[4]) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
        : "r"(w));
}
VB_DEVINL float2 kv4_f2(uint32_t halves) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&halves));
}
/* A block's scale as a number: NaN for byte 255. */
VB_DEVINL float kv4_scale_value(uint32_t byte) {
    return byte == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float(byte << 23);
}

/* ------------------------------------------------------------------ elements */
VB_DEVINL float serve_get(const float *p) { return *p; }
VB_DEVINL float serve_get(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
VB_DEVINL float serve_get(const __half *p) { return __half2float(*p); }
VB_DEVINL void serve_put(float *p, float v) { *p = v; }
VB_DEVINL void serve_put(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }
VB_DEVINL void serve_put(__half *p, float v) { *p = __float2half_rn(v); }

VB_DEVINL float2 serve_pair(uint32_t w, const float *) { return make_float2(__uint_as_float(w), 0.0f); }
VB_DEVINL float2 serve_pair(uint32_t w, const __nv_bfloat16 *) { return make_float2(vb_bf16_lo(w), vb_bf16_hi(w)); }
VB_DEVINL float2 serve_pair(uint32_t w, const __half *) { return kv4_f2(w); }
VB_DEVINL uint32_t serve_pack(float a, float b, const __nv_bfloat16 *) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
VB_DEVINL uint32_t serve_pack(float a, float b, const __half *) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

/* N values side by side; `wide`: 16-byte accesses are aligned */
template <int N, class T>
VB_DEVINL void serve_load(const T *p, bool wide, float (&x)[N]) {
    constexpr int kEach = 16 / sizeof(T);
    if (N % kEach == 0 && wide) {
#pragma unroll
        for (int i = 0; i < N / kEach; i++) {
            const uint4 w = reinterpret_cast<const uint4 *>(p)[i];
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if constexpr (sizeof(T) == 4) {
                    x[i * 4 + j] = __uint_as_float(u[j]);
                } else {
                    const float2 f = serve_pair(u[j], p);
                    x[i * 8 + 2 * j] = f.x;
                    x[i * 8 + 2 * j + 1] = f.y;
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = serve_get(p + i);
    }
}
template <int N, class T>
VB_DEVINL void serve_store(T *p, bool wide, const float (&x)[N]) {
    constexpr int kEach = 16 / sizeof(T);
    if (N % kEach == 0 && wide) {
#pragma unroll
        for (int i = 0; i < N / kEach; i++) {
            uint32_t u[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if constexpr (sizeof(T) == 4) u[j] = __float_as_uint(x[i * 4 + j]);
                else u[j] = serve_pack(x[i * 8 + 2 * j], x[i * 8 + 2 * j + 1], p);
            }
            reinterpret_cast<uint4 *>(p)[i] = make_uint4(u[0], u[1], u[2], u[3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) serve_put(p + i, x[i]);
    }
}
/* Four values side by side as they lie there, and what they are: a load whose result is not looked at yet waits for nothing. `wide`: they
 * are aligned to their size */
template <class T>
struct ServeRaw4 {
    uint32_t w[sizeof(T)];                                /* 16 bytes, or 8 */
    VB_DEVINL void none() {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); i++) w[i] = 0u;
    }
    VB_DEVINL void load(const T *p, bool wide) {
        if constexpr (sizeof(T) == 4) {
            const uint32_t *u = reinterpret_cast<const uint32_t *>(p);
            if (wide) {
                const uint4 v = *reinterpret_cast<const uint4 *>(p);
                w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = u[i];
            }
        } else {
            const uint16_t *u = reinterpret_cast<const uint16_t *>(p);
            if (wide) {
                const uint2 v = *reinterpret_cast<const uint2 *>(p);
                w[0] = v.x; w[1] = v.y;
            } else {
                w[0] = u[0] | (uint32_t)u[1] << 16;
                w[1] = u[2] | (uint32_t)u[3] << 16;
            }
        }
    }
    VB_DEVINL float4 get() const {
        if constexpr (sizeof(T) == 4) {
            return make_float4(__uint_as_float(w[0]), __uint_as_float(w[1]), __uint_as_float(w[2]), __uint_as_float(w[3]));
        } else {
            const float2 a = serve_pair(w[0], (const T *)nullptr), b = serve_pair(w[1], (const T *)nullptr);
            return make_float4(a.x, a.y, b.x, b.y);
        }
    }
};
/* Whether every row of heads begins on a 16-byte boundary. */
template <class T>
bool serve_wide(const ServeRows<T> &r) {
    constexpr long long kEach = 16 / sizeof(T);
    return ((uintptr_t)r.data & 15) == 0 && r.seq % kEach == 0 && r.row % kEach == 0 && r.head % kEach == 0;
}

/* ------------------------------------------------------------------ launchers (vb_kv4_attn.cu) */
struct Kv4Work {
    float *part, *aside;         /* partial results of key splits; sums put aside */
    unsigned *tickets, *rooms;   /* zero between calls; rooms: which places of aside are taken, one an SM */
    int *status;                 /* set where a bounded wait ran out */
    size_t part_floats;
    int n_tickets, sm_count;
};
/* Once a device, before the first call: nothing is left to be loaded inside a capture. */
int kv4_attention_load(int blocks);
int kv4_attention(const Kv4 &c, const Kv4Work &w, const vb200_kv4_attention_t &a, cudaStream_t st);

} // namespace vb

struct vb200_kv4 {
    vb::Kv4 c;
    vb::Kv4Work w;
    void *base;
    size_t bytes;
    int device, head_dim;
};

#endif

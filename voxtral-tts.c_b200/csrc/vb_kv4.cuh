/*
 * vb_kv4.cuh - what the kernels of attention over the 4-bit cache share (vb_kv4_attn.cu, vb_kv4_prompt.cu).
 */
#ifndef VB_KV4_CUH
#define VB_KV4_CUH

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

constexpr float kKv4Bias = 7.0f;              /* weights are held times 2^7 */
/* FP16 terms of a weight */
template <class T>
constexpr int kWeightTerms = std::is_same<T, __nv_bfloat16>::value ? 1 : 2;

struct Kv4Attn {
    Kv4 c;
    const int *lengths, *rows;
    int max_rows, heads, group, row_tiles, split, wide, wide_out;
    float scale;
    float *lse;
    const float *mass_in;
    float *mass_out;
    float *part;
    unsigned *tickets;
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
/* Many rows, heads up to 128 (vb_kv4_prompt.cu) */
template <class T>
int kv4_prompt(const Kv4Attn &a, const ServeRows<T> &q, const ServeRows<T> &out, cudaStream_t st);
int kv4_prompt_load(int blocks);

} // namespace vb

#endif

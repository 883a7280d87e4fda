// kvq8_attn.h -- device pieces shared by the attention kernels over the paged
// 8-bit cache: codes as fp16 operands, query rows, page numbers and scales.
#pragma once

#include "common.h"
#include "kvq8.h"

namespace hipgpt {
namespace kvq8 {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));

// Weights are kept as p * 2^(15 - lazy) relative to a running maximum m that
// moves only when a tile exceeds it by more than 2^lazy, so that O is seldom
// scaled again: fp16 then holds p up to 2^15, down to 2^-24 / 2^(15 - lazy) of
// the row's largest.  An fp32 result (two terms) keeps 4 bits more of the small
// ones than a bf16 result.
constexpr float lazy_bits(int terms) { return terms == 2 ? 4.f : 8.f; }
// V scales under this share of the largest count as this share of it.
constexpr float kMinRatio = 0x1p-40f;

// k with vs < 2^(k - 126); 0 for NaN
__device__ __forceinline__ int scale_exp(float vs) {
    const int k = (int)(__float_as_uint(vs) >> 23);
    return k < 255 ? k : 0;
}

// Two codes of word w as fp16 numbers.
template <int HI>
__device__ __forceinline__ half2v codes2(unsigned w) {
    const unsigned x = __builtin_amdgcn_perm(0x64646464u, w, HI ? 0x04030402u : 0x04010400u);
    const half2v bias = {(_Float16)1152.f, (_Float16)1152.f};
    return __builtin_bit_cast(half2v, x) - bias;
}
__device__ __forceinline__ half8 codes8(unsigned w0, unsigned w1) {
    const half2v a = codes2<0>(w0), b = codes2<1>(w0), c = codes2<0>(w1), d = codes2<1>(w1);
    return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ float lane_value(float x, int lane) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane));
}

template <class T>
__device__ __forceinline__ void load8(const T* p, float* x);
template <>
__device__ __forceinline__ void load8<float>(const float* p, float* x) {
    const floatx4 a = *reinterpret_cast<const floatx4*>(p), b = *reinterpret_cast<const floatx4*>(p + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        x[j] = a[j];
        x[4 + j] = b[j];
    }
}
template <>
__device__ __forceinline__ void load8<__bf16>(const __bf16* p, float* x) {
    const bf16x8 a = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (float)a[j];
}

// 2^e and 2^-e with x * 2^e in [2^13, 2^14) for the largest |x| of a row
// (1 where that is 0 or not finite).
__device__ __forceinline__ void row_scale(float amax, float& up, float& down) {
    const int e = (int)(__float_as_uint(amax) >> 23);  // biased exponent
    up = down = 1.f;
    if (e == 255 || amax == 0.f) return;
    const int k = min(13 - (e - 127), 126);
    up = __uint_as_float((unsigned)(127 + k) << 23);
    down = __uint_as_float((unsigned)(127 - k) << 23);
}

// Page numbers and scales of a wave's tiles t, t + step, ..., one tile a lane,
// loaded 64 tiles at a time.  A page index outside the pool reads as page 0
// with scales NaN.
struct TileMeta {
    int page;
    float ks, vs;
    __device__ __forceinline__ void load(const Cache& c, int b, int h, int t, int step, int end, int lane) {
        const int mt = t + lane * step;
        page = 0;
        ks = vs = 0.f;
        if (mt < end) {
            const int p = page_of(c, b, mt * kTile);
            page = max(p, 0);
            const int64_t at = page * c.s_page_stride + h * c.s_head_stride;
            ks = p < 0 ? __builtin_nanf("") : c.ks[at];
            vs = p < 0 ? __builtin_nanf("") : c.vs[at];
        }
    }
};

}  // namespace kvq8
}  // namespace hipgpt

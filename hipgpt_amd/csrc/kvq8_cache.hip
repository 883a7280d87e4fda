// kvq8_cache.hip -- tokens into and out of the paged 8-bit cache (kvq8.h).
//
// Append, per (page, head) and for K and V apart:
//   x    = the page's new rows (K rotated by position)
//   s'   = max(max|x| / 127, 2^-126, s if the page holds earlier tokens)
//   c    = rint(x / s'), and where s' > s the earlier codes c <- rint(c s / s')
// One workgroup owns a (page, head), keeps the page's new values in registers
// (32 a thread) between the maximum and the rounding, and so reads each row
// once.  A page with a value that is not finite gets the scale NaN, which
// stays while the page fills: what reads the page is NaN.
//
// Rotation: pair i of position p turns by p * f_i, f_i in turns as 0.64 fixed
// point, so p * f_i mod 2^64 is the exact fraction of a turn at any position;
// its upper 32 bits as fp32 are within 2^-26 turns.
#include "common.h"
#include "kernels.h"
#include "kvq8.h"

namespace hipgpt {
namespace kvq8 {

namespace {

constexpr int kUnits = 4;  // 8-value units per thread: one page of one head per workgroup

template <class T>
__device__ __forceinline__ float to_f32(T x) {
    return (float)x;
}

__device__ __forceinline__ float2 sincos_turns(uint64_t freq, int pos) {
    const int t = (int)((uint64_t)(int64_t)pos * freq >> 32);  // fraction of a turn, signed, 2^-32
    float s, c;
    sincospif((float)t * 0x1p-31f, &s, &c);
    return float2{c, s};
}

// Row d of a rotated row x (8 consecutive head dims from d0).  cs: (cos, sin)
// of the row's position per pair.
template <class T>
__device__ __forceinline__ void rotated8(const T* x, int d0, const AppendArgs& a, const float2* cs, float* y) {
    float own[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) own[j] = to_f32(x[d0 + j]);
    const int half = a.rot >> 1;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int d = d0 + j;
        y[j] = own[j];
        if (d < a.rot) {
            const bool second = a.interleaved ? (d & 1) : d >= half;
            const int i = a.interleaved ? d >> 1 : second ? d - half : d;
            const float other = a.interleaved ? own[j ^ 1] : to_f32(x[second ? d - half : d + half]);
            const float2 w = cs[i];
            y[j] = second ? fmaf(own[j], w.x, other * w.y) : fmaf(own[j], w.x, -(other * w.y));
        }
    }
}

__device__ __forceinline__ unsigned block_max(unsigned x, unsigned* red) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) x = max(x, (unsigned)__shfl_xor((int)x, m));
    const int wave = threadIdx.x >> 6, waves = (blockDim.x + 63) >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[wave] = x;
    __syncthreads();
    for (int w = 0; w < waves; ++w) x = max(x, red[w]);
    return x;
}

// Scale of a page from max|x| of its new rows (as bits: NaN above infinity
// above every number) and the scale of its earlier tokens.
__device__ __forceinline__ float page_scale(unsigned amax_bits, bool has_old, float old) {
    if (amax_bits >= 0x7f800000u) return __builtin_nanf("");
    const float s = fmaxf(__uint_as_float(amax_bits) / 127.f, kMinScale);
    if (!has_old) return s;
    return old > s || old != old ? old : s;
}

// rint(x * inv) + 128 as a byte: 2^23 * 1.5 + 128 leaves the whole number in
// the low bits, rounded to nearest even by the addition.
__device__ __forceinline__ unsigned code_of(float x, float inv) {
    return __float_as_uint(fmaf(x, inv, 12583040.f)) & 0xffu;
}
// An earlier code in the page's new, larger step (r = old / new scale).
__device__ __forceinline__ unsigned recode(unsigned u, float r) { return code_of((float)((int)u - 128), r); }

template <class T>
__device__ void append_page(const Cache& c, const AppendArgs& a, int b, int j, int h, bool is_v, float2* cs,
                            unsigned* red) {
    const Seq s = sequence(c, b);
    if (s.n == 0 || s.bad || s.len == 0) return;
    const int ps = 1 << c.lps, D = c.D, first = s.len - s.n;
    const int base = ((first >> c.lps) + j) << c.lps;  // position of the page's first token
    if (base >= s.len) return;
    const int page = page_of(c, b, base);
    if (page < 0) return;
    const int t0 = max(first - base, 0), t1 = min(s.len - base, ps);  // the page's new tokens
    const int row0 = s.row0 + base - first;                           // buffer row of page token 0 (may be < 0)
    uint8_t* codes = (is_v ? c.v : c.k) + page * c.page_stride + h * c.head_stride;
    float* sp = (is_v ? c.vs : c.ks) + page * c.s_page_stride + h * c.s_head_stride;
    const T* x = is_v ? static_cast<const T*>(a.v) + h * a.v_hs : static_cast<const T*>(a.k) + h * a.k_hs;
    const int64_t ts = is_v ? a.v_ts : a.k_ts;
    const float old = t0 > 0 ? *sp : 0.f;

    const int nt = blockDim.x, tid = threadIdx.x;
    const int units = ps * D / 8;
    float val[kUnits][8];
    unsigned amax = 0;
    if (is_v) {
        // unit (tile, q, d): tokens 32 tile + 4q..+3 and +16
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int id = tid + u * nt;
            if (id >= units) break;
            const int d = id % D, tq = id / D;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int tok = (tq >> 2) * 32 + (k >> 2) * 16 + (tq & 3) * 4 + (k & 3);
                val[u][k] = tok >= t0 && tok < t1 ? to_f32(x[(row0 + tok) * ts + d]) : 0.f;
                amax = max(amax, __float_as_uint(val[u][k]) & 0x7fffffffu);
            }
        }
    } else {
        // unit (token, 8 head dims), 32 tokens at a time for the table of angles
        const int pairs = a.freqs ? a.rot >> 1 : 0, upr = D / 8, per = 32 * upr;  // units per 32 tokens
        int u = 0;
#pragma unroll
        for (int u0 = 0; u0 < kUnits; ++u0)
#pragma unroll
            for (int k = 0; k < 8; ++k) val[u0][k] = 0.f;
        for (int sub = 0; sub < ps; sub += 32) {
            const int s0 = max(sub, t0), s1 = min(sub + 32, t1);
            if (pairs && s0 < s1) {
                __syncthreads();
                for (int i = tid; i < (s1 - s0) * pairs; i += nt) {
                    const int tok = s0 + i / pairs, p = i % pairs;
                    cs[(tok - sub) * pairs + p] = sincos_turns(a.freqs[p], base + tok);
                }
                __syncthreads();
            }
#pragma unroll
            for (int u0 = 0; u0 < kUnits; ++u0) {
                const int id = tid + u0 * nt;
                const int tok = id / upr;
                if (id < sub * upr || id >= sub * upr + per) continue;
                if (tok >= t0 && tok < t1) {
                    const T* row = x + (row0 + tok) * ts;
                    const int d0 = (id % upr) * 8;
                    if (pairs) {
                        rotated8(row, d0, a, cs + (tok - sub) * pairs, val[u0]);
                    } else {
#pragma unroll
                        for (int k = 0; k < 8; ++k) val[u0][k] = to_f32(row[d0 + k]);
                    }
#pragma unroll
                    for (int k = 0; k < 8; ++k) amax = max(amax, __float_as_uint(val[u0][k]) & 0x7fffffffu);
                }
            }
        }
        (void)u;
    }
    amax = block_max(amax, red);
    const float scale = page_scale(amax, t0 > 0, old);
    const float inv = 1.0f / scale;
    const bool grown = t0 > 0 && scale != old && old == old;
    const float r = old / scale;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const int id = tid + u * nt;
        if (id >= units) break;
        uint2 w = {0u, 0u};
        if (is_v) {
            const int d = id % D, tq = id / D;
            const int lo = (tq >> 2) * 32 + (tq & 3) * 4;  // tokens lo..lo+3 and lo+16..lo+19
            uint2* at = reinterpret_cast<uint2*>(codes + v_byte(lo, d, D));
            int fresh = 0, earlier = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int tok = lo + (k >> 2) * 16 + (k & 3);
                fresh += tok >= t0 && tok < t1;
                earlier += tok < t0;
            }
            if (fresh == 0 && !(grown && earlier)) continue;
            if (fresh < 8) w = *at;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int tok = lo + (k >> 2) * 16 + (k & 3);
                unsigned& word = k < 4 ? w.x : w.y;
                const int sh = 8 * (k & 3);
                if (tok >= t0 && tok < t1)
                    word = (word & ~(0xffu << sh)) | code_of(val[u][k], inv) << sh;
                else if (grown && tok < t0)
                    word = (word & ~(0xffu << sh)) | recode((word >> sh) & 0xffu, r) << sh;
            }
            *at = w;
        } else {
            const int upr = D / 8, tok = id / upr, d0 = (id % upr) * 8;
            uint2* at = reinterpret_cast<uint2*>(codes + k_byte(tok, d0, D));
            const bool fresh = tok >= t0 && tok < t1;
            if (!fresh && !(grown && tok < t0)) continue;
            if (!fresh) w = *at;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                unsigned& word = k < 4 ? w.x : w.y;
                const int sh = 8 * (k & 3);
                const unsigned n = fresh ? code_of(val[u][k], inv) : recode((word >> sh) & 0xffu, r);
                word = (word & ~(0xffu << sh)) | n << sh;
            }
            *at = w;
        }
    }
    if (tid == 0) *sp = scale;
}

// Queries: one pair (or one head dim past the rotated ones) per thread and
// step, read and written by the same thread, so q_out may be q.
template <class T>
__device__ void rotate_queries(const Cache& c, const AppendArgs& a, int b, int chunk, float2* cs) {
    const Seq s = sequence(c, b);
    const int i0 = chunk * 32, i1 = min(s.n, i0 + 32);
    if (i0 >= i1) return;
    const int pairs = a.freqs ? a.rot >> 1 : 0, nt = blockDim.x, tid = threadIdx.x;
    for (int i = tid; i < (i1 - i0) * pairs; i += nt)
        cs[i] = sincos_turns(a.freqs[i % pairs], max(s.len - s.n, 0) + i0 + i / pairs);
    __syncthreads();
    const int items = c.D - pairs;  // pairs, then the head dims that stay
    const int per_tok = items * a.Hq;
    const float bad = s.bad ? __builtin_nanf("") : 0.f;
    for (int i = tid; i < (i1 - i0) * per_tok; i += nt) {
        const int tok = i / per_tok, rest = i % per_tok, h = rest / items, p = rest % items;
        const T* x = static_cast<const T*>(a.q) + (s.row0 + i0 + tok) * a.q_ts + h * a.q_hs;
        T* y = static_cast<T*>(a.q_out) + (s.row0 + i0 + tok) * a.qo_ts + h * a.qo_hs;
        if (p < pairs) {
            const int d0 = a.interleaved ? 2 * p : p, d1 = a.interleaved ? d0 + 1 : p + pairs;
            const float x0 = to_f32(x[d0]), x1 = to_f32(x[d1]);
            const float2 w = cs[tok * pairs + p];
            y[d0] = (T)(fmaf(x0, w.x, -(x1 * w.y)) + bad);
            y[d1] = (T)(fmaf(x1, w.x, x0 * w.y) + bad);
        } else {
            y[p + pairs] = (T)(to_f32(x[p + pairs]) + bad);
        }
    }
}

template <class T>
__global__ __launch_bounds__(1024) void append_kernel(Cache c, AppendArgs a, int page_slots, int q_chunks) {
    extern __shared__ float2 cs[];  // [32][rot / 2] cos, sin
    __shared__ unsigned red[16];
    int id = blockIdx.x;
    const int kv = c.B * page_slots * c.H * 2;
    if (id < kv) {
        const int h = id % c.H;
        id /= c.H;
        const bool is_v = id & 1;
        id >>= 1;
        append_page<T>(c, a, id / page_slots, id % page_slots, h, is_v, cs, red);
    } else {
        id -= kv;
        rotate_queries<T>(c, a, id / q_chunks, id % q_chunks, cs);
    }
}

template <class T>
__global__ __launch_bounds__(256) void read_kernel(Cache c, ReadArgs a, int tiles) {
    int id = blockIdx.x;
    const int h = id % c.H;
    id /= c.H;
    const int b = id / tiles, tile = id % tiles;
    const Seq s = sequence(c, b);
    const int first = s.len - s.n, D = c.D, tid = threadIdx.x;
    if (s.bad) {
        for (int i = tid; i < 32 * D; i += 256) {
            const int row = tile * 32 + i / D;
            if (row >= s.n) continue;
            static_cast<T*>(a.k)[(s.row0 + row) * a.k_ts + h * a.k_hs + i % D] = (T)__builtin_nanf("");
            static_cast<T*>(a.v)[(s.row0 + row) * a.v_ts + h * a.v_hs + i % D] = (T)__builtin_nanf("");
        }
        return;
    }
    const int pos0 = ((first >> 5) + tile) << 5;  // tiles lie in one page
    if (s.n == 0 || s.len == 0 || pos0 >= s.len) return;
    const int page = page_of(c, b, pos0);
    const int64_t at = (page < 0 ? 0 : page) * c.page_stride + h * c.head_stride;
    const int64_t sat = (page < 0 ? 0 : page) * c.s_page_stride + h * c.s_head_stride;
    const float ks = page < 0 ? __builtin_nanf("") : c.ks[sat], vs = page < 0 ? __builtin_nanf("") : c.vs[sat];
    const int tb = pos0 & ((1 << c.lps) - 1);  // first token in the page
    const int64_t row0 = (int64_t)s.row0 + pos0 - first;
    for (int i = tid; i < 4 * D; i += 256) {
        const int tok = i / (D / 8), d0 = (i % (D / 8)) * 8;
        if (pos0 + tok < first || pos0 + tok >= s.len) continue;
        const uint2 w = *reinterpret_cast<const uint2*>(c.k + at + k_byte(tb + tok, d0, D));
        T* y = static_cast<T*>(a.k) + (row0 + tok) * a.k_ts + h * a.k_hs + d0;
#pragma unroll
        for (int k = 0; k < 8; ++k)
            y[k] = (T)((float)((int)(((k < 4 ? w.x : w.y) >> (8 * (k & 3))) & 0xffu) - 128) * ks);
    }
    for (int i = tid; i < 4 * D; i += 256) {
        const int q = i / D, d = i % D;
        const uint2 w = *reinterpret_cast<const uint2*>(c.v + at + v_byte(tb + 4 * q, d, D));
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int tok = (k >> 2) * 16 + 4 * q + (k & 3);
            if (pos0 + tok < first || pos0 + tok >= s.len) continue;
            static_cast<T*>(a.v)[(row0 + tok) * a.v_ts + h * a.v_hs + d] =
                (T)((float)((int)(((k < 4 ? w.x : w.y) >> (8 * (k & 3))) & 0xffu) - 128) * vs);
        }
    }
}

__global__ __launch_bounds__(256) void advance_kernel(int* lens, const int* cu, int B) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b >= B) return;
    const int64_t n = cu ? (int64_t)cu[b + 1] - cu[b] : 1;
    const int64_t len = lens[b] + (n > 0 ? n : 0);
    lens[b] = len > 0x7fffffff ? 0x7fffffff : (int)len;
}

}  // namespace

bool supported(int D, int page_size) {
    return (D == 32 || D == 64 || D == 128 || D == 256) && (page_size == 32 || page_size == 64 || page_size == 128);
}

hipError_t launch_append(const Cache& c, const AppendArgs& a, int dtype, hipStream_t s) {
    const int ps = 1 << c.lps;
    const int slots = (c.max_new + ps - 2) / ps + 1;  // pages that max_new tokens can lie in
    const int chunks = a.q ? (c.max_new + 31) / 32 : 0;
    const int64_t grid = (int64_t)c.B * slots * c.H * 2 + (int64_t)c.B * chunks;
    if (grid <= 0 || grid > 0x7fffffff) return hipErrorInvalidConfiguration;
    int nt = ps * c.D / (8 * kUnits);
    if (nt < 64) nt = 64;
    const size_t lds = a.freqs ? (size_t)32 * (a.rot / 2) * sizeof(float2) : 0;
    if (dtype == kF32)
        hipLaunchKernelGGL((append_kernel<float>), dim3((unsigned)grid), dim3(nt), lds, s, c, a, slots,
                           chunks ? chunks : 1);
    else
        hipLaunchKernelGGL((append_kernel<__bf16>), dim3((unsigned)grid), dim3(nt), lds, s, c, a, slots,
                           chunks ? chunks : 1);
    return hipGetLastError();
}

hipError_t launch_read(const Cache& c, const ReadArgs& a, int dtype, hipStream_t s) {
    const int tiles = (c.max_new + 30) / 32 + 1;
    const int64_t grid = (int64_t)c.B * tiles * c.H;
    if (grid <= 0 || grid > 0x7fffffff) return hipErrorInvalidConfiguration;
    if (dtype == kF32)
        hipLaunchKernelGGL((read_kernel<float>), dim3((unsigned)grid), dim3(256), 0, s, c, a, tiles);
    else
        hipLaunchKernelGGL((read_kernel<__bf16>), dim3((unsigned)grid), dim3(256), 0, s, c, a, tiles);
    return hipGetLastError();
}

hipError_t launch_advance(int* lens, const int* cu, int B, hipStream_t s) {
    hipLaunchKernelGGL(advance_kernel, dim3((unsigned)((B + 255) / 256)), dim3(256), 0, s, lens, cu, B);
    return hipGetLastError();
}

}  // namespace kvq8
}  // namespace hipgpt

// kvq8_cache.hip -- tokens into and out of the paged 8-bit cache (kvq8.h).
//
// Append, per (page, head) and for K and V apart:
//   x    = the page's new rows (K rotated by position)
//   s'   = max(max|x| / 127, 2^-126, s if the page holds earlier tokens)
//   c    = rint(x / s'), and where s' > s the earlier codes c <- rint(c s / s')
// A page with a value that is not finite gets the scale NaN, which stays while
// the page fills: what reads the page is NaN.
//
// Rotation: pair i of position p turns by p * f_i, f_i in turns as 0.64 fixed
// point, so p * f_i mod 2^64 is the exact fraction of a turn at any position.
//
// Both kernels read each row once and keep its values in registers between the
// maximum and the rounding.  Rows are read non-temporally: what stays near is
// the codes, which are read next (11793 tokens of 16 heads D128 read back: 33 -> 25
// us), and the append itself is 6% faster.
//   append_pages_kernel: one workgroup per page, K or V, and group of heads;
//     32 values a thread.  A thread keeps its place in the page from head to
//     head, so it forms its sines and cosines once for all the heads (K's and
//     the queries') of its group.  Bound by memory and the maximum's barriers:
//     11793 tokens of 16 + 16 heads D128 bf16 (241 MB in and out) 67 us, 3.6 TB/s
//     where a large copy reaches 4.8; 2 / 4 / 8 heads a group 67 / 67 / 68 (1: 40%
//     more), the queries in workgroups of their own 73, the next head's rows
//     requested early level, groups of 16 neighbouring head dims (lanes 32 bytes
//     apart) 7% slower.
//   append_token_kernel: one token per sequence; a wave per row.  Bound by the
//     latency of length -> page -> scale: 64 sequences, 32 + 8 heads D128 4.8 us,
//     one sequence 3.6.
// read_kernel: bound by memory, 56772 tokens of 8 heads D128 to bf16 (349 MB)
// 78 us, 4.5 TB/s; non-temporal stores 60, but what reads the rows next takes that
// much longer (and 39 -> 44 us for both at 64 MB, fp32 rows 20 -> 46 alone).
#include "common.h"
#include "kernels.h"
#include "kvq8.h"

namespace hipgpt {
namespace kvq8 {

namespace {

// cos and sin of 2 pi (pos * freq): the fraction of a turn to 32 bits, taken to
// the nearest quarter (exact), the rest |x| <= pi / 4 by the Taylor sums
// (x^11 / 11! and x^10 / 10! under 2.5e-8 there).
__device__ __forceinline__ void turn(uint64_t freq, int pos, float& c, float& s) {
    const int t = (int)((uint64_t)(int64_t)pos * freq >> 32);
    const unsigned quarter = ((unsigned)t + 0x20000000u) >> 30;
    const float x = (float)(int)((unsigned)t - (quarter << 30)) * (6.28318530717958647692f * 0x1p-32f);
    const float z = x * x;
    float a = fmaf(z, 1.f / 362880.f, -1.f / 5040.f);
    a = fmaf(z, a, 1.f / 120.f);
    a = fmaf(z, a, -1.f / 6.f);
    const float sn = fmaf(x * z, a, x);
    float b = fmaf(z, 1.f / 40320.f, -1.f / 720.f);
    b = fmaf(z, b, 1.f / 24.f);
    b = fmaf(z, b, -0.5f);
    const float cn = fmaf(z, b, 1.f);
    const float c0 = quarter & 1 ? sn : cn, s0 = quarter & 1 ? cn : sn;
    c = (quarter + 1) & 2 ? -c0 : c0;
    s = quarter & 2 ? -s0 : s0;
}

template <class T>
struct Vec;
template <>
struct Vec<float> {
    typedef float v4 __attribute__((ext_vector_type(4)));
};
template <>
struct Vec<__bf16> {
    typedef __bf16 v4 __attribute__((ext_vector_type(4)));
};

template <class T>
__device__ __forceinline__ void load4(const T* p, float* x) {
    const typename Vec<T>::v4 v = __builtin_nontemporal_load(reinterpret_cast<const typename Vec<T>::v4*>(p));
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = (float)v[j];
}
template <class T>
__device__ __forceinline__ void store4(T* p, const float* x) {
    typename Vec<T>::v4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (T)x[j];
    *reinterpret_cast<typename Vec<T>::v4*>(p) = v;
}

// rint(x * inv) + 128 as a byte: 2^23 * 1.5 + 128 leaves the whole number in
// the low bits, rounded to nearest even by the addition.
__device__ __forceinline__ unsigned code_of(float x, float inv) {
    return __float_as_uint(fmaf(x, inv, 12583040.f)) & 0xffu;
}
__device__ __forceinline__ unsigned codes4(const float* x, float inv) {
    return code_of(x[0], inv) | code_of(x[1], inv) << 8 | code_of(x[2], inv) << 16 | code_of(x[3], inv) << 24;
}
// Earlier codes in the page's new, larger step (r = old / new scale).
__device__ __forceinline__ unsigned recode4(unsigned w, float r) {
    float x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = (float)((int)(w >> (8 * k) & 0xffu) - 128);
    return codes4(x, r);
}

__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Scale of a page from max|x| of its new rows (as bits: NaN above infinity
// above every number) and the scale of its earlier tokens.
struct Scale {
    float scale, inv, r;
    bool grown;  // the earlier codes have to be rounded again, times r
    __device__ __forceinline__ Scale(unsigned amax, bool has_old, float old) {
        scale = amax >= 0x7f800000u ? __builtin_nanf("") : fmaxf(__uint_as_float(amax) / 127.f, kMinScale);
        if (has_old && (old > scale || old != old)) scale = old;
        inv = 1.0f / scale;
        grown = has_old && old == old && scale != old;
        r = old / scale;
    }
};

__device__ __forceinline__ unsigned wave_umax(unsigned x) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) x = max(x, (unsigned)__shfl_xor((int)x, m));
    return x;
}

// Rounds the codes of tokens [0, n) of a page again; one of nt threads.
__device__ void recode_page(uint8_t* codes, bool is_v, int n, int D, float r, int tid, int nt) {
    if (!is_v) {
        for (int i = tid; i < n * D / 16; i += nt) {
            uint4* p = reinterpret_cast<uint4*>(codes) + i;
            uint4 w = *p;
            *p = uint4{recode4(w.x, r), recode4(w.y, r), recode4(w.z, r), recode4(w.w, r)};
        }
        return;
    }
    // 8 bytes: tokens t .. t + 3 and t + 16 .. t + 19 of one head dim
    for (int i = tid; i < (n + 31) / 32 * (4 * D); i += nt) {
        const int t = i / (4 * D) * 32 + (i >> 5 & 3) * 4;
        uint2* p = reinterpret_cast<uint2*>(codes) + i;
        uint2 w = *p;
        const uint2 x = {recode4(w.x, r), recode4(w.y, r)};
        // bytes of tokens below n
        const int a = min(max(n - t, 0), 4), b = min(max(n - t - 16, 0), 4);
        const unsigned ma = a == 4 ? ~0u : (1u << 8 * a) - 1u, mb = b == 4 ? ~0u : (1u << 8 * b) - 1u;
        *p = uint2{(x.x & ma) | (w.x & ~ma), (x.y & mb) | (w.y & ~mb)};
    }
}

// Where a row's rotated pairs are: (2i, 2i + 1) (or none), (i, i + rot / 2) with
// rot / 2 a multiple of 8, or any other rot / 2.
enum { kPairs, kHalves, kOdd };

// 16 values of a row: head dims d0 .. d0 + 7 and d1 .. d1 + 7, so that a wave's
// loads have no gaps; values j and j + 8 (kPairs: 2i and 2i + 1) are a rotated
// pair.  With kOdd, groups hold what is left over and head dims are taken one
// by one.
template <int MODE>
struct Group {
    static constexpr bool ODD = MODE == kOdd;
    int d0, d1;  // first head dim of j < 8 and of j >= 8
    int n0, n1;  // valid ones of each (ODD)
    int pair, pair4;  // first and fifth of the eight pairs, or -1
    __device__ __forceinline__ void init(int g, int D, const AppendArgs& a) {
        n0 = n1 = 8;
        pair = pair4 = -1;
        const int half = a.rot >> 1;
        if (MODE == kPairs) {
            d0 = 8 * g;
            d1 = d0 + D / 2;
            if (a.rot) pair = d0 / 2, pair4 = d1 / 2;
        } else {
            const int ng = (half + 7) >> 3;
            if (g < ng) {
                pair = d0 = 8 * g;
                pair4 = pair + 4;
                d1 = d0 + half;
                if (ODD) n0 = n1 = min(8, half - d0);
            } else {
                d0 = a.rot + 16 * (g - ng);
                d1 = d0 + 8;
                if (ODD) {
                    n0 = min(8, max(0, D - d0));
                    n1 = min(8, max(0, D - d1));
                }
            }
        }
    }
    template <class T>
    __device__ __forceinline__ void load(const T* row, float* x) const {
        if constexpr (ODD) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] = j < n0 ? (float)row[d0 + j] : 0.f;
                x[8 + j] = j < n1 ? (float)row[d1 + j] : 0.f;
            }
        } else {
            load4(row + d0, x);
            load4(row + d0 + 4, x + 4);
            load4(row + d1, x + 8);
            load4(row + d1 + 4, x + 12);
        }
    }
    template <class T>
    __device__ __forceinline__ void store(T* row, const float* x) const {
        if constexpr (ODD) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (j < n0) row[d0 + j] = (T)x[j];
                if (j < n1) row[d1 + j] = (T)x[8 + j];
            }
        } else {
            store4(row + d0, x);
            store4(row + d0 + 4, x + 4);
            store4(row + d1, x + 8);
            store4(row + d1 + 4, x + 12);
        }
    }
    __device__ __forceinline__ void store_codes(uint8_t* row, const float* x, float inv) const {
        if constexpr (ODD) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (j < n0) row[d0 + j] = (uint8_t)code_of(x[j], inv);
                if (j < n1) row[d1 + j] = (uint8_t)code_of(x[8 + j], inv);
            }
        } else {
            *reinterpret_cast<uint2*>(row + d0) = uint2{codes4(x, inv), codes4(x + 4, inv)};
            *reinterpret_cast<uint2*>(row + d1) = uint2{codes4(x + 8, inv), codes4(x + 12, inv)};
        }
    }
    __device__ __forceinline__ void angles(const AppendArgs& a, int pos, float* c, float* s) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            c[j] = 1.f;
            s[j] = 0.f;
            const int p = j < 4 ? pair + j : pair4 + j - 4;
            if (pair >= 0 && p < (a.rot >> 1)) turn(a.freqs[p], pos, c[j], s[j]);
        }
    }
    __device__ __forceinline__ void rotate(const AppendArgs& a, float* x, const float* c, const float* s) const {
        if (pair < 0) return;
        const int half = a.rot >> 1;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // pair j: (j, j + 8) or (2j, 2j + 1)
            float& p = MODE == kPairs ? x[2 * j] : x[j];
            float& q = MODE == kPairs ? x[2 * j + 1] : x[j + 8];
            const float p0 = p, q0 = q;
            const bool on = (j < 4 ? pair + j : pair4 + j - 4) < half;
            p = on ? fmaf(p0, c[j], -(q0 * s[j])) : p0;
            q = on ? fmaf(q0, c[j], p0 * s[j]) : q0;
        }
    }
};

// Grid: (K, V) x (page slots of each sequence) x (head groups).  Threads:
// page_size * D / 32.
template <class T, int D, int MODE>
__global__ __launch_bounds__(4 * D) void append_pages_kernel(Cache c, AppendArgs a, int page_slots, int groups) {
    constexpr bool ODD = MODE == kOdd;
    constexpr int U = ODD ? 3 : 2;  // groups of 16 values per thread
    __shared__ unsigned red[2][16];
    const int tid = threadIdx.x, nt = blockDim.x, waves = (nt + 63) >> 6;
    int id = blockIdx.x;
    const int hg = id % groups;
    id /= groups;
    const bool is_v = id >= c.B * page_slots;  // last: K's workgroups, with queries, have more to do
    if (is_v) id -= c.B * page_slots;
    const int b = id / page_slots, slot = id % page_slots;
    const Seq s = sequence(c, b);
    if (s.n == 0) return;
    const int ps = 1 << c.lps;
    const bool store = !s.bad && s.len > 0;
    const int first = store ? s.len - s.n : 0;               // a bad sequence's rows count from 0
    const int base = ((first >> c.lps) + slot) << c.lps;     // position of the page's first token
    if (base >= first + s.n) return;
    const int t0 = max(first - base, 0), t1 = min(first + s.n - base, ps);  // the page's new tokens
    const int64_t row0 = (int64_t)s.row0 + base - first;     // buffer row of page token 0 (may be < 0)
    const int page = store ? page_of(c, b, base) : -1;
    const int hn = (c.H + groups - 1) / groups, h0 = hg * hn, h1 = page < 0 ? h0 : min(c.H, h0 + hn);
    int turns = 0;  // heads done, for the two reduction buffers
    auto block_max = [&](unsigned x) {
        unsigned* r = red[turns++ & 1];
        x = wave_umax(x);
        if ((tid & 63) == 0) r[tid >> 6] = x;
        __syncthreads();
        for (int w = 0; w < waves; ++w) x = max(x, r[w]);
        return x;
    };

    if (is_v) {
        // thread: 8 tokens (4q .. and 16 + 4q ..) of 4 head dims
        const int unit = tid;
        const int c4 = unit >> 1 & 3, e = unit & 1, q = unit >> 3 & 3;
        const int db = unit / 32 % (D / 32), tile = unit / D;
        const int d0 = db * 32 + e * 16 + c4 * 4, lo = tile * 32 + q * 4;
        int fresh = 0;  // bit k: token lo + 16 (k / 4) + k % 4 is new
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int tok = lo + (k >> 2) * 16 + (k & 3);
            fresh |= (tok >= t0 && tok < t1) << k;
        }
        float x[8][4];
        auto load = [&](int h) {
            const T* v = static_cast<const T*>(a.v) + h * a.v_hs + d0;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (fresh >> k & 1)
                    load4(v + (row0 + lo + (k >> 2) * 16 + (k & 3)) * a.v_ts, x[k]);
                else
                    x[k][0] = x[k][1] = x[k][2] = x[k][3] = 0.f;
            }
        };
        for (int h = h0; h < h1; ++h) {
            load(h);
            uint8_t* codes = c.v + page * c.page_stride + h * c.head_stride;
            float* sp = c.vs + page * c.s_page_stride + h * c.s_head_stride;
            const float old = t0 > 0 ? *sp : 0.f;
            unsigned amax = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) amax = max(amax, abs_bits(x[k][j]));
            const Scale sc(block_max(amax), t0 > 0, old);
            if (sc.grown) {
                recode_page(codes, true, t0, D, sc.r, tid, nt);
                __syncthreads();  // before the new tokens' bytes beside them
            }
            if (fresh) {
                uint2* at = reinterpret_cast<uint2*>(codes + v_byte(lo, d0, D));
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint2 w = {0u, 0u}, m = {0u, 0u};
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        unsigned& word = k < 4 ? w.x : w.y;
                        unsigned& mask = k < 4 ? m.x : m.y;
                        word |= code_of(x[k][j], sc.inv) << 8 * (k & 3);
                        if (fresh >> k & 1) mask |= 0xffu << 8 * (k & 3);
                    }
                    if (fresh != 0xff) {
                        const uint2 had = at[2 * j];
                        w.x = (w.x & m.x) | (had.x & ~m.x);
                        w.y = (w.y & m.y) | (had.y & ~m.y);
                    }
                    at[2 * j] = w;
                }
            }
            if (tid == 0) *sp = sc.scale;
        }
        return;
    }

    const int half = a.rot >> 1;
    const int per_row = ODD ? ((half + 7) >> 3) + ((D - a.rot + 15) >> 4) : D / 16;
    Group<MODE> gr[U];
    int tok[U];
    bool live[U];
    float cs[U][8], sn[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int g = tid + u * nt;
        tok[u] = g / per_row;
        live[u] = tok[u] >= t0 && tok[u] < t1;
        gr[u].init(g % per_row, D, a);
        if (live[u] && a.freqs) gr[u].angles(a, base + tok[u], cs[u], sn[u]);
    }
    for (int h = h0; h < h1; ++h) {
        uint8_t* codes = c.k + page * c.page_stride + h * c.head_stride;
        float* sp = c.ks + page * c.s_page_stride + h * c.s_head_stride;
        const float old = t0 > 0 ? *sp : 0.f;
        float x[U][16];
        unsigned amax = 0;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (live[u]) {
                gr[u].load(static_cast<const T*>(a.k) + (row0 + tok[u]) * a.k_ts + h * a.k_hs, x[u]);
                if (a.freqs) gr[u].rotate(a, x[u], cs[u], sn[u]);
#pragma unroll
                for (int j = 0; j < 16; ++j) amax = max(amax, abs_bits(x[u][j]));
            }
        const Scale sc(block_max(amax), t0 > 0, old);
        if (sc.grown) recode_page(codes, false, t0, D, sc.r, tid, nt);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (live[u]) gr[u].store_codes(codes + tok[u] * D, x[u], sc.inv);
        if (tid == 0) *sp = sc.scale;
    }
    if (!a.q) return;
    const int qn = (a.Hq + groups - 1) / groups, q1 = min(a.Hq, hg * qn + qn);
    for (int h = hg * qn; h < q1; ++h) {
        float x[U][16];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (live[u]) gr[u].load(static_cast<const T*>(a.q) + (row0 + tok[u]) * a.q_ts + h * a.q_hs, x[u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (live[u]) {
                if (a.freqs) gr[u].rotate(a, x[u], cs[u], sn[u]);
                if (s.bad) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) x[u][j] = __builtin_nanf("");
                }
                gr[u].store(static_cast<T*>(a.q_out) + (row0 + tok[u]) * a.qo_ts + h * a.qo_hs, x[u]);
            }
    }
}

// One token per sequence: a wave per row (K head, V head or query head), lanes
// by head dims.  Bound by the latency of length -> page -> scale.
template <class T, int D>
__global__ __launch_bounds__(256) void append_token_kernel(Cache c, AppendArgs a) {
    constexpr int E = D > 64 ? D / 64 : 1;  // head dims per lane: lane + 64 e
    const int per = 2 * c.H + (a.q ? a.Hq : 0);
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (item >= (int64_t)c.B * per) return;
    const int b = __builtin_amdgcn_readfirstlane((int)(item / per));
    const int x = __builtin_amdgcn_readfirstlane((int)(item % per));
    const int lane = threadIdx.x & 63;
    const bool on = D >= 64 || lane < D;
    const bool is_q = x >= 2 * c.H, is_v = !is_q && x >= c.H;
    const int h = is_q ? x - 2 * c.H : is_v ? x - c.H : x;
    const Seq s = sequence(c, b);
    if (s.n == 0 || (!is_q && (s.bad || s.len == 0))) return;
    const T* row = is_q   ? static_cast<const T*>(a.q) + s.row0 * a.q_ts + h * a.q_hs
                   : is_v ? static_cast<const T*>(a.v) + s.row0 * a.v_ts + h * a.v_hs
                          : static_cast<const T*>(a.k) + s.row0 * a.k_ts + h * a.k_hs;
    const int pos = s.bad || s.len == 0 ? 0 : s.len - 1;
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = on ? (float)row[lane + 64 * e] : 0.f;
    if (a.freqs && !is_v) {
        const int half = a.rot >> 1;
        float y[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int d = lane + 64 * e;
            y[e] = v[e];
            if (d < a.rot) {
                const bool second = a.interleaved ? d & 1 : d >= half;
                const float other = (float)row[a.interleaved ? d ^ 1 : second ? d - half : d + half];
                float cs, sn;
                turn(a.freqs[a.interleaved ? d >> 1 : second ? d - half : d], pos, cs, sn);
                y[e] = fmaf(v[e], cs, second ? other * sn : -(other * sn));
            }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = y[e];
    }
    if (is_q) {  // all lanes have read their pairs: q_out may be q
        T* out = static_cast<T*>(a.q_out) + s.row0 * a.qo_ts + h * a.qo_hs;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (on) out[lane + 64 * e] = (T)(s.bad ? __builtin_nanf("") : v[e]);
        return;
    }
    const int page = page_of(c, b, pos);
    if (page < 0) return;
    const int tok = pos & ((1 << c.lps) - 1);
    uint8_t* codes = (is_v ? c.v : c.k) + page * c.page_stride + h * c.head_stride;
    float* sp = (is_v ? c.vs : c.ks) + page * c.s_page_stride + h * c.s_head_stride;
    const float old = tok > 0 ? *sp : 0.f;
    unsigned amax = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) amax = max(amax, abs_bits(v[e]));
    const Scale sc(wave_umax(amax), tok > 0, old);
    if (sc.grown) {
        recode_page(codes, is_v, tok, D, sc.r, lane, 64);
        __threadfence_block();  // before the new token's bytes beside them
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int d = lane + 64 * e;
        if (on) codes[is_v ? v_byte(tok, d, D) : k_byte(tok, d, D)] = (uint8_t)code_of(v[e], sc.inv);
    }
    if (lane == 0) *sp = sc.scale;
}

// One 32-token tile of one head: D threads with 8 tokens of 4 head dims of V,
// D threads with two 16-byte pieces of K rows.
template <class T, int D>
__global__ __launch_bounds__(2 * D) void read_kernel(Cache c, ReadArgs a, int tiles) {
    int id = blockIdx.x;
    const int h = id % c.H;
    id /= c.H;
    const int b = id / tiles, tile = id % tiles;
    const Seq s = sequence(c, b);
    const int tid = threadIdx.x;
    if (s.n == 0 || (s.len == 0 && !s.bad)) return;
    const int first = s.bad ? 0 : s.len - s.n;
    const int pos0 = ((first >> 5) + tile) << 5;  // tiles lie in one page
    if (pos0 >= first + s.n) return;
    const int page = s.bad ? -1 : page_of(c, b, pos0);
    const int64_t at = (int64_t)max(page, 0) * c.page_stride + (int64_t)h * c.head_stride;
    const int64_t sat = (int64_t)max(page, 0) * c.s_page_stride + (int64_t)h * c.s_head_stride;
    const int tb = pos0 & ((1 << c.lps) - 1);  // first token in the page
    const int64_t row0 = (int64_t)s.row0 + pos0 - first;
    const int lo = max(first - pos0, 0), hi = min(first + s.n - pos0, 32);
    const bool is_v = tid >= D;
    const float sc = page < 0 ? __builtin_nanf("") : (is_v ? c.vs : c.ks)[sat];
    auto value = [&](unsigned w, int k) { return (float)((int)(w >> (8 * k) & 0xffu) - 128) * sc; };
    if (is_v) {
        const int u = tid % D;
        const int e = u & 1, c4 = u >> 1 & 3, q = u >> 3 & 3, db = u >> 5;
        const int d0 = db * 32 + e * 16 + c4 * 4;
        const uint2* p = reinterpret_cast<const uint2*>(c.v + at + v_byte(tb + 4 * q, d0, D));
        uint2 w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = p[2 * j];
        T* y = static_cast<T*>(a.v) + h * a.v_hs + d0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int tok = (k >> 2) * 16 + 4 * q + (k & 3);
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = value(k < 4 ? w[j].x : w[j].y, k & 3);
            if (tok >= lo && tok < hi) store4(y + (row0 + tok) * a.v_ts, x);
        }
        return;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int i = tid + u * D, tok = i / (D / 16), d0 = i % (D / 16) * 16;
        const uint4 w = *reinterpret_cast<const uint4*>(c.k + at + k_byte(tb + tok, d0, D));
        const unsigned ws[4] = {w.x, w.y, w.z, w.w};
        T* y = static_cast<T*>(a.k) + (row0 + tok) * a.k_ts + h * a.k_hs + d0;
        if (tok >= lo && tok < hi) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float x[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] = value(ws[j], k);
                store4(y + 4 * j, x);
            }
        }
    }
}

__global__ __launch_bounds__(256) void advance_kernel(int* lens, const int* cu, int B) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b >= B) return;
    if (lens[b] < 0) return;  // a slot without a sequence
    const int64_t n = cu ? (int64_t)cu[b + 1] - cu[b] : 1;
    const int64_t len = lens[b] + (n > 0 ? n : 0);
    lens[b] = len > 0x7fffffff ? 0x7fffffff : (int)len;
}

template <class T, int D>
hipError_t append_d(const Cache& c, const AppendArgs& a, hipStream_t s) {
    if (c.max_new == 1) {
        const int64_t rows = (int64_t)c.B * (2 * (int64_t)c.H + (a.q ? a.Hq : 0));
        if (rows > 0x7fffffff) return hipErrorInvalidConfiguration;
        hipLaunchKernelGGL((append_token_kernel<T, D>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, c, a);
        return hipGetLastError();
    }
    const int ps = 1 << c.lps;
    const int slots = (c.max_new + ps - 2) / ps + 1;  // pages that max_new tokens can lie in
    // Heads of a workgroup share their sines and cosines; fewer workgroups than
    // ~2 per CU and role would leave CUs idle.
    const int64_t pages = (int64_t)(c.T + ps - 1) / ps + c.B;
    int per = 4;
    while (per > 1 && pages * ((c.H + per - 1) / per) < 512) per /= 2;
    const int groups = (c.H + per - 1) / per;
    const int64_t grid = (int64_t)c.B * slots * 2 * groups;
    if (grid <= 0 || grid > 0x7fffffff) return hipErrorInvalidConfiguration;
    const dim3 nt(ps * D / 32 < 64 ? 64 : ps * D / 32);  // a whole wave: idle lanes have no token
    auto kern = !a.rot || a.interleaved ? append_pages_kernel<T, D, kPairs>
                : a.rot % 16            ? append_pages_kernel<T, D, kOdd>
                                        : append_pages_kernel<T, D, kHalves>;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), nt, 0, s, c, a, slots, groups);
    return hipGetLastError();
}

template <class T, int D>
hipError_t read_d(const Cache& c, const ReadArgs& a, hipStream_t s) {
    const int tiles = (c.max_new + 30) / 32 + 1;
    const int64_t grid = (int64_t)c.B * tiles * c.H;
    if (grid <= 0 || grid > 0x7fffffff) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((read_kernel<T, D>), dim3((unsigned)grid), dim3(2 * D), 0, s, c, a, tiles);
    return hipGetLastError();
}

}  // namespace

bool supported(int D, int page_size) {
    return (D == 32 || D == 64 || D == 128 || D == 256) && (page_size == 32 || page_size == 64 || page_size == 128);
}

hipError_t launch_append(const Cache& c, const AppendArgs& a, int dtype, hipStream_t s) {
    const bool f = dtype == kF32;
    switch (c.D) {
        case 32: return f ? append_d<float, 32>(c, a, s) : append_d<__bf16, 32>(c, a, s);
        case 64: return f ? append_d<float, 64>(c, a, s) : append_d<__bf16, 64>(c, a, s);
        case 128: return f ? append_d<float, 128>(c, a, s) : append_d<__bf16, 128>(c, a, s);
        case 256: return f ? append_d<float, 256>(c, a, s) : append_d<__bf16, 256>(c, a, s);
        default: return hipErrorInvalidValue;
    }
}

hipError_t launch_read(const Cache& c, const ReadArgs& a, int dtype, hipStream_t s) {
    const bool f = dtype == kF32;
    switch (c.D) {
        case 32: return f ? read_d<float, 32>(c, a, s) : read_d<__bf16, 32>(c, a, s);
        case 64: return f ? read_d<float, 64>(c, a, s) : read_d<__bf16, 64>(c, a, s);
        case 128: return f ? read_d<float, 128>(c, a, s) : read_d<__bf16, 128>(c, a, s);
        case 256: return f ? read_d<float, 256>(c, a, s) : read_d<__bf16, 256>(c, a, s);
        default: return hipErrorInvalidValue;
    }
}

hipError_t launch_advance(int* lens, const int* cu, int B, hipStream_t s) {
    hipLaunchKernelGGL(advance_kernel, dim3((unsigned)((B + 255) / 256)), dim3(256), 0, s, lens, cu, B);
    return hipGetLastError();
}

}  // namespace kvq8
}  // namespace hipgpt

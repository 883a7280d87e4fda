// kvq8_attn.hip -- attention over the paged 8-bit cache (kvq8.h).
//
// For query row r (token i of a sequence's new ones, query head g of those
// that share a cached head) and the keys j <= its position:
//   s_j = scale * ks(page j) * sum_d q_d c_jd
//   o   = sum_j p_j vs(page j) c'_jd / sum_j p_j,   p_j = exp(s_j - max s)
//
// Products run on the fp16 matrix cores: a code is exact in fp16 (1024 + u is
// the bit pattern 0x6400 | u, minus 1152 leaves c), and the other operand is
// given as one or two fp16 terms.
//   * q is scaled by a power of two so that its largest element is in
//     [2^13, 2^14): a bf16 q is then one exact term (what is 2^-37 of the
//     largest element or less rounds), an fp32 q two terms, off by 2^-23 of
//     each element at most.
//   * p, kept within 2^15 of the row's running maximum, is one term for a
//     bf16 result (off by 2^-12 of itself) and two for an fp32 result.
// With 16-row tiles the second terms cost nothing: they are columns of their
// own in the same product (8 rows a tile instead of 16), and the two halves
// are added once per score and once at the end.
//
// S^T = K Q^T (16 tokens x 16 rows): lane (c, q) of the accumulator holds
// tokens 4q..4q+3 of row c; two such products make the 32-token B operand of
// O^T = V^T P^T without leaving registers, the cache's V tiles being in that
// token order.  V scales are applied to p relative to the largest met so far,
// one number for all rows, so a page costs one multiplication per score.
#include "common.h"
#include "kernels.h"
#include "kvq8_attn.h"

namespace hipgpt {
namespace kvq8 {

namespace {

constexpr int NW = 4;            // waves per workgroup
constexpr float kPShift = 15.f;  // p is kept as p * 2^15: fp16 then holds 2^-39 .. 1

__device__ __forceinline__ float xor8_add(float x) {  // + the lane 8 places away in its row of 16
    const int y = __builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xf, 0xf, false);
    return x + __int_as_float(y);
}
// over the four lanes that hold one column
__device__ __forceinline__ float col_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float col_sum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// Raw codes of one 32-token tile of one head.
template <int D>
struct Tile {
    static constexpr int KL = D / 64 ? D / 64 : 1;  // 16-byte loads of a 16-token K sub-tile (one of 8 bytes at D = 32)
    uint4 k[2][KL];
    uint4 v[D / 32];
};

template <int D>
__device__ __forceinline__ void load_tile(Tile<D>& t, const uint8_t* kp, const uint8_t* vp, int c, int q, int lane) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        if constexpr (D == 32) {
            const uint2 w = *reinterpret_cast<const uint2*>(kp + (s * 16 + c) * D + q * 8);
            t.k[s][0] = uint4{w.x, w.y, 0u, 0u};
        } else {
#pragma unroll
            for (int i = 0; i < D / 64; ++i)
                t.k[s][i] = *reinterpret_cast<const uint4*>(kp + (s * 16 + c) * D + i * 64 + q * 16);
        }
    }
#pragma unroll
    for (int i = 0; i < D / 32; ++i) t.v[i] = *reinterpret_cast<const uint4*>(vp + i * 1024 + lane * 16);
}

// First head dim of the 8 that lane quarter q holds in k-step s of Q K^T.
template <int D>
__device__ __forceinline__ int q_dim(int s, int q) {
    return D == 32 ? q * 8 : (s >> 1) * 64 + q * 16 + (s & 1) * 8;
}

// One workgroup: 16 / TERMS rows of one (sequence, cached head), one split of
// its keys; the four waves take every fourth 32-token tile and are joined in
// LDS.  TERMS: columns per row (2: q and p as two fp16 terms).
template <int D, int TERMS, class TI, class TO>
__global__ __launch_bounds__(NW * 64) void attn_rows_kernel(Cache c, AttnArgsQ8 a, int row_blocks) {
    constexpr int RPB = 16 / TERMS;  // rows per block
    __shared__ float s_m[NW][16], s_l[NW][16], s_ref[NW];
    __shared__ __attribute__((aligned(16))) float s_o[NW][16][D + 4];

    int id = blockIdx.x;
    const int rb = id % row_blocks;
    id /= row_blocks;
    const int h = id % c.H;
    id /= c.H;
    const int b = id % c.B, split = id / c.B;
    const int G = a.Hq / c.H;
    const Seq s = sequence(c, b);
    const int rows = s.n * G, r0 = rb * RPB;
    if (r0 >= rows) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, q4 = lane >> 4;

    const int first = s.len - s.n;
    const int row = min(r0 + col % RPB, rows - 1);  // columns past the last row repeat it
    const int lim = s.bad ? 0 : first + row / G + 1;  // keys that the row sees
    const int top = s.bad ? 0 : first + min(r0 + RPB - 1, rows - 1) / G + 1;
    const int tiles_all = (top + kTile - 1) / kTile;
    const int per = (tiles_all + a.nsplit - 1) / a.nsplit;
    const int tile0 = split * per, tile1 = min(tiles_all, tile0 + per);

    // the query as the B operand: column = row (and term)
    half8 qv[D / 32];
    float sc;  // of a raw score, without the page's scale
    {
        const TI* qp = static_cast<const TI*>(a.q) + (int64_t)(s.row0 + row / G) * a.q_ts + (h * G + row % G) * a.q_hs;
        float x[D / 32][8], amax = 0.f, up, down;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            load8(qp + q_dim<D>(i, q4), x[i]);
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[i][j]));
        }
        row_scale(col_max(amax), up, down);
        sc = down * a.qscale;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y = x[i][j] * up;
                const _Float16 hi = (_Float16)y;
                qv[i][j] = TERMS == 2 && col >= 8 ? (_Float16)(y - (float)hi) : hi;
            }
    }

    floatx4 o[D / 16];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[i] = floatx4{0.f, 0.f, 0.f, 0.f};
    float m = kMaxInit, l = 0.f, ref = 0.f;

    TileMeta meta;
    int cnt = 0;
    for (int t = tile0 + wave; t < tile1; t += NW, ++cnt) {
        if ((cnt & 63) == 0) meta.load(c, b, h, t, NW, tile1, lane);
        const int page = __builtin_amdgcn_readlane(meta.page, cnt & 63);
        const float ks = lane_value(meta.ks, cnt & 63), vs = lane_value(meta.vs, cnt & 63);
        const int tok = (t * kTile) & ((1 << c.lps) - 1);
        const int64_t at = (int64_t)page * c.page_stride + (int64_t)h * c.head_stride + tok * D;
        Tile<D> tl;
        load_tile<D>(tl, c.k + at, c.v + at, col, q4, lane);

        floatx4 sv[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            sv[u] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                const uint4 w = tl.k[u][i >> 1];
                const half8 kv = (i & 1) ? codes8(w.z, w.w) : codes8(w.x, w.y);
                sv[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv, qv[i], sv[u], 0, 0, 0);
            }
        }
        float f = sc * ks, mt = kMaxInit;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (TERMS == 2) sv[u][r] = xor8_add(sv[u][r]);
                sv[u][r] = t * kTile + u * 16 + q4 * 4 + r < lim ? sv[u][r] * f : kNegInf;
                mt = fmaxf(mt, sv[u][r]);
            }
        mt = col_max(mt);
        const float mn = fmaxf(m, mt);
        float alpha = fast_exp2(m - mn);
        m = mn;
        l *= alpha;
        if (vs > ref) {
            alpha *= ref / vs;
            ref = vs;
        }
        if (__any(alpha != 1.f)) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[i] *= alpha;
        }
        const float ratio = ref > 0.f ? vs / ref : vs;
        half8 pv;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float p = fast_exp2(sv[u][r] - m + kPShift);
                l += p;
                const float w = sv[u][r] == kNegInf ? 0.f : p * ratio;
                const _Float16 hi = (_Float16)w;
                pv[u * 4 + r] = TERMS == 2 && col >= 8 ? (_Float16)(w - (float)hi) : hi;
            }
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            o[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(tl.v[i].x, tl.v[i].y), pv, o[2 * i], 0, 0, 0);
            o[2 * i + 1] =
                __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(tl.v[i].z, tl.v[i].w), pv, o[2 * i + 1], 0, 0, 0);
        }
    }

    // join the waves: true O = o * ref, on the common maximum
    l = col_sum(l);
    if (q4 == 0) {
        s_m[wave][col] = m;
        s_l[wave][col] = l;
    }
    if (lane == 0) s_ref[wave] = ref;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) *reinterpret_cast<floatx4*>(&s_o[wave][col][i * 16 + q4 * 4]) = o[i];
    __syncthreads();
    for (int i = tid; i < RPB * D; i += NW * 64) {
        const int rr = i / D, d = i % D;
        if (r0 + rr >= rows) continue;
        float M = kMaxInit, L = 0.f, O = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, s_m[w][rr]);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float e = fast_exp2(s_m[w][rr] - M);
            float x = s_o[w][rr][d];
            if (TERMS == 2) x += s_o[w][rr + 8][d];
            L = fmaf(s_l[w][rr], e, L);
            O = fmaf(x * s_ref[w], e, O);
        }
        O = L > 0.f || L != L ? O / L : 0.f;  // no visible key: zeros
        if (s.bad) L = O = __builtin_nanf("");
        const int tok = (r0 + rr) / G, g = (r0 + rr) % G;
        const int64_t orow = s.row0 + tok;
        if (a.nsplit == 1) {
            static_cast<TO*>(a.o)[orow * a.o_ts + (h * G + g) * a.o_hs + d] = (TO)O;
        } else {
            const int64_t slot = (orow * a.Hq + h * G + g) * a.nsplit + split;
            if (d == 0) {
                a.ws[2 * slot] = M;
                a.ws[2 * slot + 1] = L;
            }
            a.ws[2 * (int64_t)c.T * a.Hq * a.nsplit + slot * D + d] = O;
        }
    }
}

// Joins the splits of rows: O = sum_s O_s L_s 2^(m_s - M) / sum_s L_s 2^(m_s - M).
// D / 4 lanes (four head dims each) and PAR of them side by side per row: the
// split rows of one row are loaded PAR at a time, since each load waits for
// memory that another XCD wrote.  A workgroup of 256 takes 256 / (PAR D / 4) rows.
template <int D, int PAR, class TO>
__global__ __launch_bounds__(256) void attn_join_kernel(Cache c, AttnArgsQ8 a) {
    constexpr int LP = D / 4;            // lanes per split row
    constexpr int TPR = LP * PAR;        // threads per row
    constexpr int RPW = 256 / TPR;       // rows per workgroup
    __shared__ __attribute__((aligned(16))) float s_o[PAR > 1 ? 256 : 1][4];
    __shared__ float s_l[PAR > 1 ? 256 : 1];
    const int tid = threadIdx.x, sub = tid % LP, par = tid / LP % PAR;
    const int64_t item = (int64_t)blockIdx.x * RPW + tid / TPR;  // (sequence, token, head)
    const int h = (int)(item % a.Hq);
    const int64_t bi = item / a.Hq;
    bool live = bi < (int64_t)c.B * c.max_new;
    int64_t row = 0;
    if (live) {
        const Seq q = sequence(c, (int)(bi / c.max_new));
        live = bi % c.max_new < q.n;
        row = q.row0 + bi % c.max_new;
    }
    floatx4 O = {0.f, 0.f, 0.f, 0.f};
    float L = 0.f;
    if (live) {
        const int64_t slot = (row * a.Hq + h) * a.nsplit;
        const float2* ml = reinterpret_cast<const float2*>(a.ws) + slot;
        const float* po = a.ws + 2 * (int64_t)c.T * a.Hq * a.nsplit + slot * D + sub * 4;
        float M = kMaxInit;
        for (int s = 0; s < a.nsplit; ++s) M = fmaxf(M, ml[s].x);
#pragma unroll 4
        for (int s = par; s < a.nsplit; s += PAR) {
            const float2 x = ml[s];
            const float w = x.y * fast_exp2(x.x - M);
            const floatx4 v = *reinterpret_cast<const floatx4*>(po + (int64_t)s * D);
            L += w;
            if (w != 0.f) O += w * v;
        }
    }
    if constexpr (PAR > 1) {
        *reinterpret_cast<floatx4*>(s_o[tid]) = O;
        s_l[tid] = L;
        __syncthreads();
        if (par != 0) return;
#pragma unroll
        for (int g = 1; g < PAR; ++g) {
            O += *reinterpret_cast<const floatx4*>(s_o[tid + g * LP]);
            L += s_l[tid + g * LP];
        }
    }
    if (!live) return;
    TO* op = static_cast<TO*>(a.o) + row * a.o_ts + h * a.o_hs + sub * 4;
#pragma unroll
    for (int v = 0; v < 4; ++v) op[v] = (TO)(L > 0.f || L != L ? O[v] / L : 0.f);
}

template <int D, int PAR, class TO>
hipError_t launch_join_t(const Cache& c, const AttnArgsQ8& a, hipStream_t s) {
    constexpr int RPW = 256 / (D / 4 * PAR);
    const int64_t grid = ((int64_t)c.B * c.max_new * a.Hq + RPW - 1) / RPW;
    if (grid > 0x7fffffff) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((attn_join_kernel<D, PAR, TO>), dim3((unsigned)grid), dim3(256), 0, s, c, a);
    return hipGetLastError();
}

template <int D, class TO>
hipError_t launch_join(const Cache& c, const AttnArgsQ8& a, hipStream_t s) {
    // few splits: a row needs no help; many: as many lanes as a workgroup has
    if (a.nsplit <= 4) return launch_join_t<D, 1, TO>(c, a, s);
    return launch_join_t<D, 1024 / D, TO>(c, a, s);
}

template <int D, int TERMS, class TI, class TO>
hipError_t launch_rows(const Cache& c, const AttnArgsQ8& a, hipStream_t s) {
    const int rpb = 16 / TERMS;
    const int64_t row_blocks = ((int64_t)c.max_new * (a.Hq / c.H) + rpb - 1) / rpb;
    const int64_t grid = row_blocks * c.H * c.B * a.nsplit;
    if (grid <= 0 || grid > 0x7fffffff) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((attn_rows_kernel<D, TERMS, TI, TO>), dim3((unsigned)grid), dim3(NW * 64), 0, s, c, a,
                       (int)row_blocks);
    return hipGetLastError();
}

template <int D>
hipError_t launch_dim(const Cache& c, const AttnArgsQ8& a, int dtype, int out_dtype, hipStream_t s) {
        hipError_t e;
    if (tiles_for(c.max_new, a.Hq / c.H)) return launch_tiles(c, a, dtype, out_dtype, s);
    if (dtype == kF32)
        e = launch_rows<D, 2, float, float>(c, a, s);
    else if (out_dtype == kF32)
        e = launch_rows<D, 2, __bf16, float>(c, a, s);
    else
        e = launch_rows<D, 1, __bf16, __bf16>(c, a, s);
    if (e != hipSuccess || a.nsplit == 1) return e;
    return out_dtype == kF32 ? launch_join<D, float>(c, a, s) : launch_join<D, __bf16>(c, a, s);
}

}  // namespace

// Whether so many rows of one cached head take the 128-row blocks.
bool tiles_for(int max_new, int G) { return (int64_t)max_new * G > 32; }

int attn_splits(int B, int T, int max_new, int Hq, int Hkv, int D, int max_len) {
    const int64_t G = Hq / Hkv;
    if (tiles_for(max_new, (int)G)) {
        const int64_t blocks = Hkv * (T * G / 128 + B);  // row blocks, at most
        return blocks < tile_shares(D) && max_len >= 1024 ? tile_shares(D) : 1;
    }
    const int64_t wgs = Hkv * B * ((max_new * G + 15) / 16);
    int n = 1;
    while (n < 256 && wgs * n <= 512 && max_len / (2 * n) >= 256) n *= 2;
    return n;
}

size_t attn_workspace(int T, int max_new, int Hq, int Hkv, int D, int nsplit) {
    if (nsplit <= 1) return 0;
    if (tiles_for(max_new, Hq / Hkv)) return tile_workspace(D, nsplit);
    return (size_t)T * Hq * nsplit * (size_t)(D + 2) * sizeof(float);
}

hipError_t launch_attn(const Cache& c, const AttnArgsQ8& a, int dtype, int out_dtype, hipStream_t s) {
    switch (c.D) {
        case 32: return launch_dim<32>(c, a, dtype, out_dtype, s);
        case 64: return launch_dim<64>(c, a, dtype, out_dtype, s);
        case 128: return launch_dim<128>(c, a, dtype, out_dtype, s);
        case 256: return launch_dim<256>(c, a, dtype, out_dtype, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace kvq8
}  // namespace hipgpt

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
//   * p, relative to a running maximum of the row, is one term for a bf16
//     result (off by 2^-12 of itself) and two for an fp32 result.
// With 16-row tiles the second terms cost nothing: they are columns of their
// own in the same product (8 rows a tile instead of 16), and the two halves
// are added once per score and once at the end.
//
// Bound by memory: a copy of the kernel that only loads the codes takes as long.
// 64 sequences of 512 .. 8192 keys, 32/8 heads D128 bf16 (572 MB) 107 us + 5 us
// join, 5.3 TB/s; 2 of 65537 and 131072 keys 78 + 6 us; 64 of up to 2048, 12 heads
// D64 fp32 (101 MB) 26 us, where the longest sequence decides (loads alone 22);
// one of 333 keys 6.1 us, three loads' latency and the launch.  Equal shares of
// all keys in place of splits (as kvq8_tiles.hip has them) lost: 118 + 7, 85 + 5
// and 37 us.
//
// S^T = K Q^T (16 tokens x 16 rows): lane (c, q) of the accumulator holds
// tokens 4q..4q+3 of row c; two such products make the 32-token B operand of
// O^T = V^T P^T without leaving registers, the cache's V tiles being in that
// token order.  A V scale is applied to p relative to a power of two above the
// largest met so far, in the exponent; the row sum takes it out again once a
// tile.
#include "common.h"
#include "kernels.h"
#include "kvq8_attn.h"

namespace hipgpt {
namespace kvq8 {

namespace {

constexpr int NW = 4;  // waves per workgroup (8: 572 MB above 108 -> 115 us, one of 1000 keys 10.3 -> 9.1)

__device__ __forceinline__ float xor8_add(float x) {  // + the lane 8 places away in its row of 16
    const int y = __builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xf, 0xf, false);
    return x + __int_as_float(y);
}
// over the four lanes (16 apart) that hold one column
__device__ __forceinline__ float col_max(float x) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float col_sum(float x) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Raw codes of one 32-token tile of one head.  Non-temporal: a decode step
// reads them once (572 MB of 32/8 heads D128: 119 -> 108 us).
__device__ __forceinline__ uint4 load16(const uint8_t* p) {
    const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
    return uint4{v[0], v[1], v[2], v[3]};
}
template <int D>
struct Tile {
    static constexpr int KL = D / 64 ? D / 64 : 1;  // 16-byte loads of a 16-token K sub-tile (one of 8 bytes at D = 32)
    uint4 k[2][KL];
    uint4 v[D / 32];
    float ks, vs;
    __device__ __forceinline__ void load(const uint8_t* kp, const uint8_t* vp, int c, int q, int lane) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            if constexpr (D == 32) {
                const uint2 w = *reinterpret_cast<const uint2*>(kp + (s * 16 + c) * D + q * 8);
                k[s][0] = uint4{w.x, w.y, 0u, 0u};
            } else {
#pragma unroll
                for (int i = 0; i < D / 64; ++i) k[s][i] = load16(kp + (s * 16 + c) * D + i * 64 + q * 16);
            }
        }
#pragma unroll
        for (int i = 0; i < D / 32; ++i) v[i] = load16(vp + i * 1024 + lane * 16);
    }
};

// First head dim of the 8 that lane quarter q holds in k-step s of Q K^T.
template <int D>
__device__ __forceinline__ int q_dim(int s, int q) {
    return D == 32 ? q * 8 : (s >> 1) * 64 + q * 16 + (s & 1) * 8;
}

// One workgroup: 16 / TERMS rows of one (sequence, cached head), one split of
// its keys; the four waves take every fourth 32-token tile and are joined in
// LDS.  TERMS: columns per row (2: q and p as two fp16 terms).
template <int D, int TERMS, class TI, class TO>
__global__ __launch_bounds__(NW * 64, D <= 64 ? 4 : D == 128 ? 3 : 2) void attn_rows_kernel(Cache c, AttnArgsQ8 a,
                                                                                           int row_blocks) {
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
    const int low = s.bad ? 0 : first + r0 / G + 1;   // ... the block's first row
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
    float m = kMaxInit, l = 0.f;
    int kref = 0;

    // Two tiles' codes in registers (D <= 128): while one is multiplied the
    // wave's next is on its way.
    TileMeta meta;
    Tile<D> tl[2];
    int cnt = 0;
    auto fetch = [&](Tile<D>& to, int t) {
        if ((cnt & 63) == 0) meta.load(c, b, h, t, NW, tile1, lane);
        const int page = __builtin_amdgcn_readlane(meta.page, cnt & 63);
        to.ks = lane_value(meta.ks, cnt & 63);
        to.vs = lane_value(meta.vs, cnt & 63);
        ++cnt;
        const int64_t at = (int64_t)page * c.page_stride + (int64_t)h * c.head_stride +
                           ((t * kTile) & ((1 << c.lps) - 1)) * D;
        to.load(c.k + at, c.v + at, col, q4, lane);
    };
    auto process = [&](const Tile<D>& tl, int t) {
        const float f = sc * tl.ks, vs_now = tl.vs;
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
        const int left = lim - t * kTile - 4 * q4;  // score (u, r) is seen: 16 u + r below this
        const bool edge = (t + 1) * kTile > low;     // some row does not see some token
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (TERMS == 2) sv[u][r] = xor8_add(sv[u][r]);
        if (edge) {
            asm volatile("");  // a branch: most tiles have no edge
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (16 * u + r >= left) sv[u][r] = kNegInf;
        }
        float mt = sv[0][0];
#pragma unroll
        for (int r = 1; r < 8; ++r) mt = fmaxf(mt, sv[r >> 2][r & 3]);
        mt = col_max(mt) * f;  // NaN (a scale of NaN or 0) moves nothing
        float alpha = 1.f;
        if (mt > m + lazy_bits(TERMS)) {
            alpha = fast_exp2(m - mt);
            m = mt;
        }
        l *= alpha;
        const int k = scale_exp(vs_now);
        if (k > kref) {
            alpha = __builtin_amdgcn_ldexpf(alpha, kref - k);
            kref = k;
        }
        if (__any(alpha != 1.f)) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[i] *= alpha;
        }
        const float ratio = fmaxf(__builtin_amdgcn_ldexpf(vs_now, 126 - kref), kMinRatio);
        const float e0 = (15.f - lazy_bits(TERMS) - m) + (vs_now == vs_now ? __builtin_amdgcn_logf(ratio) : vs_now);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) sv[u][r] = fast_exp2(fmaf(sv[u][r], f, e0));
        if (edge) {  // also where a scale of 0 or NaN made NaN of what a row does not see
            asm volatile("");
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (16 * u + r >= left) sv[u][r] = 0.f;
        }
        float sum = 0.f;
        half8 pv;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                sum += sv[u][r];
                const _Float16 hi = (_Float16)sv[u][r];
                pv[u * 4 + r] = TERMS == 2 && col >= 8 ? (_Float16)(sv[u][r] - (float)hi) : hi;
            }
        l = fmaf(sum, __builtin_amdgcn_rcpf(ratio), l);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            o[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(tl.v[i].x, tl.v[i].y), pv, o[2 * i], 0, 0, 0);
            o[2 * i + 1] =
                __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(tl.v[i].z, tl.v[i].w), pv, o[2 * i + 1], 0, 0, 0);
        }
    };
    if constexpr (D <= 128) {
        if (tile0 + wave < tile1) fetch(tl[0], tile0 + wave);
        for (int t = tile0 + wave; t < tile1; t += 2 * NW) {
            if (t + NW < tile1) fetch(tl[1], t + NW);
            process(tl[0], t);
            if (t + NW >= tile1) break;
            if (t + 2 * NW < tile1) fetch(tl[0], t + 2 * NW);
            process(tl[1], t + NW);
        }
    } else {  // no registers for a second tile
        for (int t = tile0 + wave; t < tile1; t += NW) {
            fetch(tl[0], t);
            process(tl[0], t);
        }
    }

    // join the waves: O = o * (V reference), on the common maximum
    l = col_sum(l);
    if (q4 == 0) {
        s_m[wave][col] = m;
        s_l[wave][col] = l;
    }
    if (lane == 0) s_ref[wave] = __builtin_amdgcn_ldexpf(1.f, kref - 126);
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
    if (tiles_for(c.B, c.max_new, a.Hq, c.H, out_dtype)) return launch_tiles(c, a, dtype, out_dtype, s);
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

// 16-row tiles (8 with an fp32 result) that the rows of one cached head fill.
static int64_t row_tiles(int max_new, int G, int out_dtype) {
    const int rpb = out_dtype == kF32 ? 8 : 16;
    return ((int64_t)max_new * G + rpb - 1) / rpb;
}

// Whether the rows take the 128-row blocks.  One 16-row tile reads the codes
// once and needs no LDS; several read them again each, which pays only while
// they leave most CUs idle.  us, 16-row tiles / 128-row blocks, 8 heads D128
// bf16, 8 | 16 | 32 | 48 rows: 64 sequences of 2048-4096 keys 73 / 120 | 77 / 119 |
// 153 / 119 | 219 / 135, 4 of 4096-8192 21 / 40 | 22 / 41 | 32 / 42 | 45 / 46; fp32,
// 8 | 16 | 24 | 32 rows: 77 / 142 | 153 / 142 | 221 / 143 | 289 / 142 and 21 / 46 |
// 33 / 47 | 45 / 48 | 53 / 49.
bool tiles_for(int B, int max_new, int Hq, int Hkv, int out_dtype) {
    const int64_t n = row_tiles(max_new, Hq / Hkv, out_dtype);
    return n > 3 || (n > 1 && (int64_t)B * Hkv * n > 256);
}

int attn_splits(int B, int T, int max_new, int Hq, int Hkv, int D, int out_dtype, int max_len) {
    if (max_len <= 1024) return 1;
    if (tiles_for(B, max_new, Hq, Hkv, out_dtype)) {
        // shares where whole blocks are fewer than the device holds at once (1289
        // rows of 32/8 heads behind 4-8k keys: 311 us whole in two splits, 236 in
        // shares; 1024 blocks of 2048 keys: 108 us whole, 152 in shares)
        const int64_t blocks = Hkv * (T * (int64_t)(Hq / Hkv) / 128 + B);  // at most
        return blocks < tile_shares(D) ? tile_shares(D) : 1;
    }
    const int64_t wgs = Hkv * B * row_tiles(max_new, Hq / Hkv, out_dtype);
    // One workgroup per CU at least, none with fewer than 256 keys (the join is
    // a launch of ~3 us: 1000 keys of 12 heads D64 10.5 us whole, 10.8 in two),
    // and two per CU where whole rows are so long that the longest of them
    // decides (64 sequences of 512 .. 8192 keys, 8 heads D128: 113 -> 109 us).
    // More splits lose: 2 sequences of 131072 and 65537 keys 83 / 83 / 87 / 96 us
    // at 16 / 32 / 64 / 128.
    int n = 1;
    while (n < 256 && max_len / (2 * n) >= 256 &&
           (wgs * n < 256 || (wgs * n <= 512 && max_len / n >= 8192)))
        n *= 2;
    return n;
}

size_t attn_workspace(int B, int T, int max_new, int Hq, int Hkv, int D, int out_dtype, int nsplit) {
    if (nsplit <= 1) return 0;
    if (tiles_for(B, max_new, Hq, Hkv, out_dtype)) return tile_workspace(D, nsplit);
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

// kvq8_tiles.hip -- attention of a chunk of new tokens over the paged 8-bit
// cache (kvq8.h): many query rows per cached head.  Formulas and the fp16
// operands are those of kvq8_attn.hip; here the products are 32x32x16 and the
// codes become fp16 once per workgroup, in LDS.
//
// What bounds it: matrix and vector work of a SIMD's waves hardly overlap on
// this chip, so a wave costs their sum.  At D = 128, bf16 in and out, 64 tokens x
// 32 rows are 32 MFMAs (1024 cycles) and ~280 vector instructions, 32 of them
// exponentials (~1450): 512 equal workgroups, two a CU, take 2.7 us per stage
// pair (790 TFLOP/s) where that sum is 2.1.  fp32 in and out doubles the MFMAs.
// Measured: 4 prompts of 2048 tokens, 16 heads D128 bf16 105 us (655 TFLOP/s);
// 8 of 1024, 12 heads D64 fp32 43 us.  128 rows a workgroup: the codes' way to
// fp16 costs 72 of the 280, shared by its four waves; eight waves (256 rows)
// measured level at D = 128 and 10% slower at D = 64, whose codes are half.  One
// tile's products set between the next one's exponentials: 114 us instead of 105.
//
// A workgroup holds 4 waves x 32 rows (token i, query head g, in the order
// i * G + g, so that the heads that share a cached head share its tiles) and
// walks the keys 64 at a time: codes of the next 64 are in flight to registers
// while the current ones are multiplied from LDS (two buffers, one barrier).
//   S^T = K Q^T: lane (c, h) holds 16 tokens of row c.  K rows are taken in
//     the order that makes register r token 4 kq(r / 4, h) + r % 4 of the tile,
//     kq = h + 2 (r / 8) + 4 (r / 4 % 2): registers 8s .. 8s+7 are then the 8
//     tokens that the cache's V tile keeps together for lane quarter 2s + h,
//     so that P^T is the B operand of O^T = V^T P^T as it stands.
//   The V scale relative to a power of two above the largest met so far rides
//     in the exponent of p; the row sum takes it out again once per tile.
#include <type_traits>

#include "common.h"
#include "fa_common.h"
#include "kernels.h"
#include "kvq8_attn.h"

namespace hipgpt {
namespace kvq8 {

namespace {

using fa::halves_sum;

constexpr int TW = 4;              // waves
constexpr int ROWS = TW * 32;      // query rows per workgroup
constexpr int STAGE = 64;          // tokens per LDS buffer

template <int D>
struct Stage {
    static constexpr int KP = D + 8;  // halfs between K rows
    _Float16 k[STAGE * KP];
    _Float16 v[STAGE * D];
};

// Codes of one stage on their way from memory: 16-byte units, K then V.
template <int D>
struct Flight {
    static constexpr int N = D >= 64 ? D / 64 : 1;
    uint4 k[N], v[N];
};

__device__ __forceinline__ half8 load_half8(const _Float16* p) { return *reinterpret_cast<const half8*>(p); }

// Stages of row block rb of sequence b (0: it has no such rows; a sequence
// whose length is bad has one stage without tokens, for its NaN rows).
__device__ __forceinline__ int block_stages(const Cache& c, int G, int b, int rb) {
    const Seq s = sequence(c, b);
    const int rows = s.n * G, r0 = rb * ROWS;
    if (r0 >= rows) return 0;
    const int top = s.bad ? 0 : s.len - s.n + min(r0 + ROWS - 1, rows - 1) / G + 1;
    return max(1, (top + STAGE - 1) / STAGE);
}

// Part of a row block's keys: stages s0 .. s1 - 1.  slot < 0: all of them, the
// result goes to o; else to that slot of the workspace.
struct Piece {
    int b, h, rb, s0, s1, slot;
};

// Workspace of shared row blocks: a join item per share, then per slot (two a
// share) and row (m, l, scale of O, -), then O / l, fp32, or fp16 in units of
// the V reference where the result is bf16.
__device__ __forceinline__ float* slot_head(float* ws, int shares, int slot) {
    return ws + 4 * (int64_t)shares + (int64_t)slot * ROWS * 4;
}
template <int D>
__device__ __forceinline__ float* slot_rows(float* ws, int shares, int slot) {
    return slot_head(ws, shares, 2 * shares) + (int64_t)slot * ROWS * D;
}

template <int D, int TQ, int TP, class TI, class TO>
__device__ __forceinline__ void run_piece(const Cache& c, const AttnArgsQ8& a, const Piece& pc, Stage<D>* st) {
    using St = Stage<D>;
    const int b = pc.b, h = pc.h;
    const int G = a.Hq / c.H;
    const Seq s = sequence(c, b);
    const int rows = s.n * G, r0 = pc.rb * ROWS;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, hf = lane >> 5;

    const int first = s.len - s.n;
    const int w0 = r0 + wave * 32;                  // the wave's first row
    const int row = min(w0 + col, rows - 1);        // columns past the last row repeat it
    const int tok = row / G;
    const int lim = s.bad ? 0 : first + tok + 1;    // keys that the row sees
    const int wlo = s.bad ? 0 : first + min(w0, rows - 1) / G + 1;         // ... the wave's first row
    const int whi = s.bad || w0 >= rows ? 0 : first + min(w0 + 31, rows - 1) / G + 1;  // ... its last
    const int top = s.bad ? 0 : first + min(r0 + ROWS - 1, rows - 1) / G + 1;
    const int stage0 = pc.s0, stage1 = s.bad ? stage0 : pc.s1;
    const int tile_end = (top + kTile - 1) / kTile;  // tiles past it have no page

    half8 qv[TQ][D / 16];
    float sc;
    {
        const TI* qp = static_cast<const TI*>(a.q) + (int64_t)(s.row0 + tok) * a.q_ts + (h * G + row % G) * a.q_hs +
                       hf * (D / 2);
        float amax = 0.f, up, down;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
            float x[8];
            load8(qp + 8 * j, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[i]));
        }
        row_scale(fmaxf(amax, xor32(amax)), up, down);
        sc = down * a.qscale;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
            float x[8];
            load8(qp + 8 * j, x);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = x[i] * up;
                qv[0][j][i] = (_Float16)y;
                if (TQ == 2) qv[TQ - 1][j][i] = (_Float16)(y - (float)qv[0][j][i]);
            }
        }
    }

    floatx16 o[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
    float m = kMaxInit, l = 0.f;
    int kref = 0;

    TileMeta meta;
    Flight<D> fl;
    int meta_at = 2 * stage0 - 64;  // first tile that `meta` holds
    // page and scales of tile t; called with t rising
    auto meta_for = [&](int t) {
        if (t - meta_at >= 64) {
            meta_at = t;
            meta.load(c, b, h, t, 1, tile_end, lane);
        }
        return t - meta_at;
    };
    // a stage's two tiles lie in one page or two; units of 16 bytes, 2 D per tile
    auto load_stage = [&](int sg) {
        const int i0 = meta_for(2 * sg);  // even: both tiles of a stage are held together
#pragma unroll
        for (int i = 0; i < Flight<D>::N; ++i) {
            const int unit = i * (TW * 64) + tid;
            const int u = __builtin_amdgcn_readfirstlane(unit / (2 * D));
            if (D < 64 && u > 1) continue;
            const int t = 2 * sg + u;
            const int page = __builtin_amdgcn_readlane(meta.page, i0 + u);
            const int64_t at = (int64_t)page * c.page_stride + (int64_t)h * c.head_stride +
                               ((t * kTile) & ((1 << c.lps) - 1)) * D;
            const int off = unit % (2 * D) * 16;
            fl.k[i] = *reinterpret_cast<const uint4*>(c.k + at + off);
            fl.v[i] = *reinterpret_cast<const uint4*>(c.v + at + off);
        }
    };
    auto store_stage = [&](St& to) {
#pragma unroll
        for (int i = 0; i < Flight<D>::N; ++i) {
            const int unit = i * (TW * 64) + tid;
            if (D < 64 && unit >= 4 * D) continue;
            const int krow = unit * 16 / D, kd = unit * 16 % D;
            half8* kp = reinterpret_cast<half8*>(to.k + krow * St::KP + kd);
            kp[0] = codes8(fl.k[i].x, fl.k[i].y);
            kp[1] = codes8(fl.k[i].z, fl.k[i].w);
            // V: head dims c and 16 + c of a lane quarter's tokens -> [quarter][head dim]
            half8* vp = reinterpret_cast<half8*>(to.v + (unit >> 4) * 256 + (unit & 15) * 8);
            vp[0] = codes8(fl.v[i].x, fl.v[i].y);
            vp[16] = codes8(fl.v[i].z, fl.v[i].w);
        }
    };
    // lane's K row of a tile: MFMA row c holds token 4 kq + c % 4
    const int rq = col >> 2;
    const int krow = 4 * (2 * (rq >> 2) + (rq & 1) + 4 * ((rq >> 1) & 1)) + (col & 3);

    float minus_one = -1.f;
    asm("" : "+s"(minus_one));
    float cur_ks[2] = {0.f, 0.f}, cur_vs[2] = {0.f, 0.f};
    if (stage0 < stage1) {
        load_stage(stage0);
        store_stage(st[0]);
    }
    for (int sg = stage0; sg < stage1; ++sg) {
        __syncthreads();
        const St& now = st[(sg - stage0) & 1];
        {
            const int i0 = meta_for(2 * sg);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                cur_ks[u] = lane_value(meta.ks, i0 + u);
                cur_vs[u] = lane_value(meta.vs, i0 + u);
            }
        }
        if (sg + 1 < stage1) load_stage(sg + 1);
        const int tb = sg * STAGE;  // the stage's first token
        if (tb < whi) {
            const bool edge = tb + STAGE > wlo;  // some row does not see some token
            const int left = lim - tb - 4 * hf;  // a register's token is seen: its place below this
            auto place = [](int u, int r) { return 32 * u + 16 * ((r >> 2) & 1) + 8 * (r >> 3) + (r & 3); };
            const float f[2] = {sc * cur_ks[0], sc * cur_ks[1]};
            floatx16 sv[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
                for (int r = 0; r < 16; ++r) sv[u][r] = 0.f;
                const _Float16* kp = now.k + (u * kTile + krow) * St::KP + hf * (D / 2);
#pragma unroll
                for (int j = 0; j < D / 16; ++j) {
                    const half8 kf = load_half8(kp + 8 * j);
                    sv[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qv[0][j], sv[u], 0, 0, 0);
                    if (TQ == 2) sv[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qv[TQ - 1][j], sv[u], 0, 0, 0);
                }
            }
            if (edge) {
                asm volatile("");  // a branch: most stages have no edge
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (place(u, r) >= left) sv[u][r] = kNegInf;
            }
            // a scale of NaN or 0 gives NaN here, which fmaxf leaves out
            const float mt = fmaxf(fa::tile_max(sv[0]) * f[0], fa::tile_max(sv[1]) * f[1]);
            // V scale: a power of two 2^(kref - 126) above every one met is taken out of O
            const int k = max(scale_exp(cur_vs[0]), scale_exp(cur_vs[1]));
            float alpha = 1.f;
            if (mt > m + lazy_bits(TP)) {
                alpha = fast_exp2(m - mt);
                m = mt;
            }
            l *= alpha;
            if (k > kref) {
                alpha = __builtin_amdgcn_ldexpf(alpha, kref - k);
                kref = k;
            }
            if (__any(alpha != 1.f)) {
#pragma unroll
                for (int i = 0; i < D / 32; ++i) o[i] *= alpha;
            }
            float ratio[2], e0[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float vs = cur_vs[u];
                ratio[u] = fmaxf(__builtin_amdgcn_ldexpf(vs, 126 - kref), kMinRatio);
                e0[u] = (15.f - lazy_bits(TP) - m) + (vs == vs ? __builtin_amdgcn_logf(ratio[u]) : vs);
#pragma unroll
                for (int r = 0; r < 16; ++r) sv[u][r] = fast_exp2(fmaf(sv[u][r], f[u], e0[u]));
            }
            // a scale of 0 or NaN: not for rows that do not see it
            if (edge && __any(!(f[0] > 0.f) || !(f[1] > 0.f) || !(e0[0] < kInf) || !(e0[1] < kInf))) {
                asm volatile("");
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (place(u, r) >= left) sv[u][r] = 0.f;
            }
            half8 pv[TP][4];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float sum = fa::kSumInit;
#pragma unroll
                for (int r = 0; r < 16; ++r) sum += sv[u][r];
                l = fmaf(sum, __builtin_amdgcn_rcpf(ratio[u]), l);
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    const float2v x = {sv[u][r], sv[u][r + 1]};
                    const half2v hi = __builtin_convertvector(x, half2v);
                    half8& ph = pv[0][2 * u + (r >> 3)];
                    ph[r & 7] = hi[0];
                    ph[(r & 7) + 1] = hi[1];
                    if (TP == 2) {
                        // what is left: one mixed-precision fma each (minus_one is not a
                        // constant to the compiler, which would convert and subtract)
                        const float2v y = {fmaf((float)hi[0], minus_one, x[0]), fmaf((float)hi[1], minus_one, x[1])};
                        const half2v lo = __builtin_convertvector(y, half2v);
                        half8& pl = pv[TP - 1][2 * u + (r >> 3)];
                        pl[r & 7] = lo[0];
                        pl[(r & 7) + 1] = lo[1];
                    }
                }
            }
            const _Float16* vp = now.v + lane * 8;
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const half8 vf = load_half8(vp + (j >> 1) * (kTile * D) + i * 1024 + (j & 1) * 512);
                    o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pv[0][j], o[i], 0, 0, 0);
                    if (TP == 2) o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pv[TP - 1][j], o[i], 0, 0, 0);
                }
        }
        if (sg + 1 < stage1) store_stage(st[(sg + 1 - stage0) & 1]);
    }

    if (w0 + col >= rows) return;
    l = halves_sum(l);
    float norm = l > 0.f ? 1.f / l : 0.f;  // no visible key: zeros
    if (l != l || s.bad) norm = l = __builtin_nanf("");
    const float unit = __builtin_amdgcn_ldexpf(1.f, kref - 126);
    // register r of block i: head dim 32 i + 8 (r / 4) + 4 hf + r % 4
    if (pc.slot < 0) {
        norm *= unit;
        TO* op = static_cast<TO*>(a.o) + (int64_t)(s.row0 + tok) * a.o_ts + (h * G + row % G) * a.o_hs + 4 * hf;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) op[i * 32 + 8 * (r >> 2) + (r & 3)] = (TO)(o[i][r] * norm);
    } else {
        const int wr = wave * 32 + col;
        if (hf == 0)
            *reinterpret_cast<floatx4*>(slot_head(a.ws, a.nsplit, pc.slot) + 4 * wr) =
                floatx4{m, l, TP == 1 ? unit : 1.f, 0.f};
        if (TP == 2) norm *= unit;
        using W = std::conditional_t<TP == 1, _Float16, float>;
        W* op = reinterpret_cast<W*>(slot_rows<D>(a.ws, a.nsplit, pc.slot)) + wr * D + 4 * hf;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) op[i * 32 + 8 * (r >> 2) + (r & 3)] = (W)(o[i][r] * norm);
    }
}

// One workgroup per row block of a (sequence, head), over all its keys.
template <int D, int TQ, int TP, class TI, class TO>
__global__ __launch_bounds__(TW * 64, D <= 128 ? 2 : 1) void attn_tiles_kernel(Cache c, AttnArgsQ8 a, int row_blocks) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    // Longest rows first over all (sequence, head) pairs, so that the last
    // workgroups to start are short; with B H a multiple of 8 a pair stays on
    // one XCD (workgroups go to the XCDs in turn) and its tiles in that L2.
    const int BH = c.B * c.H, bh = blockIdx.x % BH;
    Piece pc;
    pc.h = bh % c.H;
    pc.b = bh / c.H;
    pc.rb = row_blocks - 1 - blockIdx.x / BH;
    pc.s0 = 0;
    pc.s1 = block_stages(c, a.Hq / c.H, pc.b, pc.rb);
    pc.slot = -1;
    if (pc.s1 == 0) return;
    run_piece<D, TQ, TP, TI, TO>(c, a, pc, reinterpret_cast<Stage<D>*>(smem));
}

// ---- equal shares of the work
// Few row blocks with many keys leave CUs idle or paired unevenly, so there the
// stages of all row blocks (heads, then sequences, then row blocks) are laid
// end to end and cut into a.nsplit equal shares, one workgroup each.  A row
// block that lies in one share is written as above; of the others each share
// writes its part to the workspace (slot 2w + 1 where the block begins in share
// w, 2w where it goes on), and a second kernel joins them.  Lengths are on the
// device, so every workgroup sums them up by itself.
constexpr int kMinShare = 4;  // stages
constexpr int kPlan = TW * 64;    // threads

struct Plan {
    int64_t wave_sum[TW];
    int64_t at;      // first stage of the item found
    int item, n;     // the item, its stages
};

struct Shares {
    int chunk;
    int64_t per_head, total, share;  // stages: more than 2^31 in a prompt of 4 M tokens
    int64_t my_pre, my_sum;
    // Items are (sequence, row block); thread t sums items [t * chunk, ...).
    __device__ __forceinline__ void init(const Cache& c, int G, int row_blocks, int count, Plan& pl) {
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        const int items = c.B * row_blocks;
        chunk = items / kPlan + 1;
        my_sum = 0;
        for (int64_t i = (int64_t)tid * chunk, e = min((int64_t)items, i + chunk); i < e; ++i)
            my_sum += block_stages(c, G, (int)(i / row_blocks), (int)(i % row_blocks));
        int64_t inc = my_sum;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t x = __shfl_up((long long)inc, d);
            if (lane >= d) inc += x;
        }
        if (lane == 63) pl.wave_sum[wave] = inc;
        __syncthreads();
        my_pre = inc - my_sum;
        per_head = 0;
#pragma unroll
        for (int w = 0; w < TW; ++w) {
            if (w < wave) my_pre += pl.wave_sum[w];
            per_head += pl.wave_sum[w];
        }
        total = per_head * c.H;
        share = max((total + count - 1) / count, (int64_t)kMinShare);
    }
    // The item that holds stage p of its head: pl.found, for all threads.
    __device__ __forceinline__ void find(const Cache& c, int G, int row_blocks, int64_t p, Plan& pl) const {
        __syncthreads();
        if (p >= my_pre && p < my_pre + my_sum) {
            int64_t at = my_pre;
            int i = threadIdx.x * chunk, n = block_stages(c, G, i / row_blocks, i % row_blocks);
            while (p >= at + n) {
                at += n;
                ++i;
                n = block_stages(c, G, i / row_blocks, i % row_blocks);
            }
            pl.item = i;
            pl.at = at;
            pl.n = n;
        }
        __syncthreads();
    }
};

template <int D, int TQ, int TP, class TI, class TO>
__global__ __launch_bounds__(TW * 64, D <= 128 ? 2 : 1) void attn_shares_kernel(Cache c, AttnArgsQ8 a, int row_blocks) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    __shared__ Plan pl;
    const int G = a.Hq / c.H;
    const int w = xcd_remap(blockIdx.x, gridDim.x);  // neighbouring shares, often of one head, on one XCD
    Shares sh;
    sh.init(c, G, row_blocks, a.nsplit, pl);
    int64_t p = w * sh.share;
    const int64_t end = min(sh.total, p + sh.share);
    int4 join = {0, 0, 0, -1};  // (sequence, head, row block, last share) of a block that begins here and goes on
    while (p < end) {
        const int h = (int)(p / sh.per_head);
        const int64_t in_head = p % sh.per_head;
        sh.find(c, G, row_blocks, in_head, pl);
        const int item = __builtin_amdgcn_readfirstlane(pl.item), n = __builtin_amdgcn_readfirstlane(pl.n);
        Piece pc;
        pc.b = item / row_blocks;
        pc.h = h;
        pc.rb = item % row_blocks;
        pc.s0 = __builtin_amdgcn_readfirstlane((int)(in_head - pl.at));
        pc.s1 = (int)min((int64_t)n, pc.s0 + (end - p));
        pc.slot = pc.s0 > 0 ? 2 * w : pc.s1 < n ? 2 * w + 1 : -1;
        if (pc.slot & 1 && pc.slot > 0) join = {pc.b, h, pc.rb, (int)((p + n - 1) / sh.share)};
        run_piece<D, TQ, TP, TI, TO>(c, a, pc, reinterpret_cast<Stage<D>*>(smem));
        p += pc.s1 - pc.s0;
    }
    if (threadIdx.x == 0) reinterpret_cast<int4*>(a.ws)[w] = join;
}

// Joins the parts of the row block that begins in share w and goes on after it:
// O = sum_s O_s L_s 2^(m_s - M) / sum_s L_s 2^(m_s - M).  Four workgroups per
// share; D / 4 lanes per row, several rows and four parts a thread in flight,
// since each load waits for memory that another XCD wrote (and 16 times as
// many, smaller workgroups took 18 us to launch where these take 8).
template <int D, int TP, class TO>
__global__ __launch_bounds__(256) void attn_shares_join_kernel(Cache c, AttnArgsQ8 a) {
    constexpr int LP = D / 4, RP = 256 / LP, NR = RP < 32 ? 32 / RP : 1, PARTS = 4;
    using W = std::conditional_t<TP == 1, _Float16, float>;
    typedef W W4 __attribute__((ext_vector_type(4)));
    const int w = blockIdx.x >> 2, rr0 = (blockIdx.x & 3) * 32 + threadIdx.x / LP;
    const int4 item = reinterpret_cast<const int4*>(a.ws)[w];
    if (item.w < 0) return;
    const int G = a.Hq / c.H, sub = threadIdx.x % LP;
    const Seq s = sequence(c, item.x);
    const int rows = s.n * G, row0 = item.z * ROWS;
    if (row0 + (int)(blockIdx.x & 3) * 32 >= rows) return;
    float M[NR], L[NR];
    floatx4 O[NR];
#pragma unroll
    for (int k = 0; k < NR; ++k) {
        M[k] = kMaxInit;
        L[k] = 0.f;
        O[k] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    for (int i0 = w; i0 <= item.w; i0 += PARTS) {
        floatx4 hd[NR][PARTS];
        W4 x[NR][PARTS];
#pragma unroll
        for (int j = 0; j < PARTS; ++j) {
            const int i = min(i0 + j, item.w), slot = i == w ? 2 * w + 1 : 2 * i;
            const float* hp = slot_head(a.ws, a.nsplit, slot);
            const W* xp = reinterpret_cast<const W*>(slot_rows<D>(a.ws, a.nsplit, slot));
#pragma unroll
            for (int k = 0; k < NR; ++k) {
                const int rr = min(rr0 + k * RP, rows - 1 - row0);  // rows past the last have no part
                hd[k][j] = *reinterpret_cast<const floatx4*>(hp + 4 * rr);
                x[k][j] = *reinterpret_cast<const W4*>(xp + rr * D + sub * 4);
            }
        }
#pragma unroll
        for (int k = 0; k < NR; ++k) {
            float mn = M[k];
#pragma unroll
            for (int j = 0; j < PARTS; ++j) mn = fmaxf(mn, hd[k][j][0]);
            const float e0 = fast_exp2(M[k] - mn);
            M[k] = mn;
            L[k] *= e0;
            O[k] *= e0;
#pragma unroll
            for (int j = 0; j < PARTS; ++j) {
                const float e1 = i0 + j <= item.w ? hd[k][j][1] * fast_exp2(hd[k][j][0] - mn) : 0.f;
                L[k] += e1;
                if (e1 != 0.f) {
                    const float e2 = e1 * hd[k][j][2];
#pragma unroll
                    for (int v = 0; v < 4; ++v) O[k][v] = fmaf((float)x[k][j][v], e2, O[k][v]);
                }
            }
        }
    }
#pragma unroll
    for (int k = 0; k < NR; ++k) {
        const int row = row0 + rr0 + k * RP;
        if (row >= rows) break;
        TO* op = static_cast<TO*>(a.o) + (int64_t)(s.row0 + row / G) * a.o_ts + (item.y * G + row % G) * a.o_hs +
                 sub * 4;
#pragma unroll
        for (int v = 0; v < 4; ++v) op[v] = (TO)(L[k] > 0.f || L[k] != L[k] ? O[k][v] / L[k] : 0.f);
    }
}

template <int D, int TQ, int TP, class TI, class TO>
hipError_t launch_tiles_t(const Cache& c, const AttnArgsQ8& a, hipStream_t s) {
    constexpr size_t lds = 2 * sizeof(Stage<D>);
    const int64_t row_blocks = ((int64_t)c.max_new * (a.Hq / c.H) + ROWS - 1) / ROWS;
    const bool shared = a.nsplit > 1;
    auto kern = shared ? attn_shares_kernel<D, TQ, TP, TI, TO> : attn_tiles_kernel<D, TQ, TP, TI, TO>;
    const int64_t grid = shared ? a.nsplit : row_blocks * c.H * c.B;
    if (row_blocks * c.B > 0x7fffffff || grid <= 0 || grid > 0x7fffffff) return hipErrorInvalidConfiguration;
    if (lds > 64 * 1024) {
        const hipError_t e =
            hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(TW * 64), lds, s, c, a, (int)row_blocks);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !shared) return e;
    hipLaunchKernelGGL((attn_shares_join_kernel<D, TP, TO>), dim3((unsigned)grid * 4), dim3(256), 0, s, c, a);
    return hipGetLastError();
}

template <int D>
hipError_t launch_tiles_d(const Cache& c, const AttnArgsQ8& a, int dtype, int out_dtype, hipStream_t s) {
    if (dtype == kF32) return launch_tiles_t<D, 2, 2, float, float>(c, a, s);
    if (out_dtype == kF32) return launch_tiles_t<D, 1, 2, __bf16, float>(c, a, s);
    return launch_tiles_t<D, 1, 1, __bf16, __bf16>(c, a, s);
}

}  // namespace

// One share per workgroup that the device holds at once: 256 CUs with two of
// them each (registers at D = 128, LDS), one at D = 256.
int tile_shares(int D) { return D == 256 ? 256 : 512; }

size_t tile_workspace(int D, int shares) {
    return (size_t)shares * (4 + 2 * ROWS * (4 + D)) * sizeof(float);
}

hipError_t launch_tiles(const Cache& c, const AttnArgsQ8& a, int dtype, int out_dtype, hipStream_t s) {
    switch (c.D) {
        case 32: return launch_tiles_d<32>(c, a, dtype, out_dtype, s);
        case 64: return launch_tiles_d<64>(c, a, dtype, out_dtype, s);
        case 128: return launch_tiles_d<128>(c, a, dtype, out_dtype, s);
        case 256: return launch_tiles_d<256>(c, a, dtype, out_dtype, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace kvq8
}  // namespace hipgpt

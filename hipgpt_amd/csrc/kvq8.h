// kvq8.h -- the paged 8-bit key/value cache: layout, bounds and the argument
// structs that its kernels share.
//
// A page holds `1 << lps` (32, 64 or 128) tokens of one sequence, for every
// head.  Codes are bytes u = c + 128, c a whole number in [-127, 127]; one
// fp32 scale per (page, head) for K and one for V; the value is c * scale.
//   K: [token][D] in a (page, head).
//   V: tiles of 32 tokens, each in the order in which a 16x16x32 MFMA takes
//      it as its A operand (rows = head dims, k = tokens): a lane (c, q)
//      reads 16 bytes that hold, for head dims 32*db + c and 32*db + 16 + c,
//      tokens 4q..4q+3 and 16+4q..16+4q+3 -- the tokens whose scores that
//      lane holds after two 16-token products.  One wave load of 64 x 16
//      bytes is 1 KB without gaps.
// The functions below are plain C++ (host and device), so their bounds are
// checked on the host as well.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace hipgpt {
namespace kvq8 {

constexpr int kTile = 32;        // tokens per V tile
constexpr int kMaxLen = 0x7fffff00;  // tokens of a sequence: a tile past it is still an int
constexpr int kMaxSplits = 1024;  // of the keys, or shares
// Smallest scale: codes of values under it stay within [-127, 127] and its
// reciprocal is finite.
constexpr float kMinScale = 1.17549435e-38f;  // 2^-126

// The cache pools and one batch of sequences over them.
struct Cache {
    uint8_t* k;
    uint8_t* v;
    float* ks;
    float* vs;
    int64_t page_stride, head_stride;    // bytes, of k and v
    int64_t s_page_stride, s_head_stride;  // floats, of ks and vs
    int num_pages, lps, H, D;
    const int* table;  // [B][max_pages] page of each `1 << lps` tokens
    int64_t t_stride;
    int max_pages;
    const int* lens;  // [B] tokens, the new ones included
    const int* cu;    // [B + 1] rows of the new tokens, or null: row b, one each
    int B, T, max_new;
};

// Sequence b of a batch: its new tokens are rows row0 .. row0 + n - 1 of the
// packed buffers and positions len - n .. len - 1.  len == 0 with a row (cu
// null) is an empty slot: nothing to store, no key to see.
struct Seq {
    int n, row0, len;
    bool bad;  // more rows than max_new, or a length outside the table: rows are NaN, nothing is stored
};

__host__ __device__ inline Seq sequence(const Cache& a, int b) {
    Seq s;
    s.row0 = a.cu ? a.cu[b] : b;
    const int64_t end = a.cu ? (int64_t)a.cu[b + 1] : (int64_t)b + 1;
    // rows outside the packed buffers: none of them is touched
    s.n = s.row0 >= 0 && end > s.row0 && end <= a.T ? (int)(end - s.row0) : 0;
    s.len = a.lens[b];
    s.bad = s.n > a.max_new || (s.len < s.n && (a.cu || s.len < 0)) || s.len > kMaxLen ||
            (int64_t)s.len > ((int64_t)a.max_pages << a.lps);
    if (s.n > a.max_new) s.n = a.max_new;
    return s;
}

// Page that holds position pos of sequence b; -1 if the table names none.
__host__ __device__ inline int page_of(const Cache& a, int b, int pos) {
    const int p = a.table[(int64_t)b * a.t_stride + (pos >> a.lps)];
    return p >= 0 && p < a.num_pages ? p : -1;
}

// Byte of (token, head dim) inside a (page, head).
__host__ __device__ inline int k_byte(int tok, int d, int D) { return tok * D + d; }
__host__ __device__ inline int v_byte(int tok, int d, int D) {
    const int t = tok & 31;
    return (tok >> 5) * (32 * D) + (d >> 5) * 1024 + ((t >> 2) & 3) * 256 + (d & 15) * 16 + ((d >> 4) & 1) * 8 +
           (t >> 4) * 4 + (t & 3);
}

// What the append takes beside the cache: new rows in the input dtype, element
// (row, head, d) at X[row * ts + head * hs + d].
struct AppendArgs {
    const void* q;  // may be null: no queries to rotate
    void* q_out;
    const void* k;
    const void* v;
    int64_t q_ts, q_hs, qo_ts, qo_hs, k_ts, k_hs, v_ts, v_hs;
    int Hq;
    const uint64_t* freqs;  // turns per position of each pair, 0.64 fixed point; null: no rotation
    int rot;                // rotated head dims, even
    int interleaved;        // pairs (2i, 2i + 1) instead of (i, i + rot / 2)
};

struct ReadArgs {
    void* k;
    void* v;
    int64_t k_ts, k_hs, v_ts, v_hs;
};

struct AttnArgsQ8 {
    const void* q;
    void* o;
    int64_t q_ts, q_hs, o_ts, o_hs;
    int Hq;
    float qscale;  // softmax scale * log2(e)
    int nsplit;
    float* ws;  // nsplit > 1
};

bool supported(int D, int page_size);
hipError_t launch_append(const Cache& c, const AppendArgs& a, int dtype, hipStream_t s);
hipError_t launch_read(const Cache& c, const ReadArgs& a, int dtype, hipStream_t s);
hipError_t launch_advance(int* lens, const int* cu, int B, hipStream_t s);
// Attention of any number of rows.  Few rows per cached head (launch_rows in
// kvq8_attn.hip) split the keys of each 16-row tile nsplit ways; more rows
// (launch_tiles) take 128-row blocks, whole with nsplit 1, else as nsplit equal
// shares of all their keys.
bool tiles_for(int B, int max_new, int Hq, int Hkv, int out_dtype);
int attn_splits(int B, int T, int max_new, int Hq, int Hkv, int D, int out_dtype, int max_len);
size_t attn_workspace(int B, int T, int max_new, int Hq, int Hkv, int D, int out_dtype, int nsplit);
hipError_t launch_attn(const Cache& c, const AttnArgsQ8& a, int dtype, int out_dtype, hipStream_t s);
hipError_t launch_tiles(const Cache& c, const AttnArgsQ8& a, int dtype, int out_dtype, hipStream_t s);
int tile_shares(int D);
size_t tile_workspace(int D, int shares);

}  // namespace kvq8
}  // namespace hipgpt

// cache_attn.cuh -- what the two attention kernels over the paged 8-bit cache
// share: cache_attn.cu (a few queries) and cache_attn_tc.cu (many).
//
//     S = q k^T sm_scale,  P = softmax(S over the tokens a query sees),  O = P V
//
// with k = code * 2^(u - 127) and v likewise.  Query t of stream b sees the
// tokens below min(lens[b], limits[b][t]); a query that sees none gives
// zeros.  Query heads that share a key/value head are rows of one tile: row
// r of (stream, key/value head) is query r / group, head r % group of its
// group.
#pragma once
#include <climits>

#include "cache.cuh"
#include "tcgen05.cuh"

namespace ress {
namespace cache {

using namespace tc;

struct AttnArgs {
    const uint16_t *q;  // bf16
    long long q_sb, q_st, q_sh;
    void *out;
    long long o_sb, o_st, o_sh;
    int out_bf16;
    int Tq, group, rows;  // rows = Tq * group
    Pages K, V;
    const int32_t *table, *lens, *limits;
    long long table_stride;
    int table_width, n_pages;
    float scale_log2;  // sm_scale * log2(e)
    int32_t *status;
    // cache_attn_tc.cu, where the pages are split over CTAs: partial results and arrival counters
    float *partial;
    int32_t *arrived;
};

// Tokens that the queries of stream b may see at most.
__device__ __forceinline__ int stream_len(const AttnArgs &a, int b) {
    const int len = a.lens[b];
    const long long cap = (long long)a.table_width * PAGE;
    return len < 0 ? 0 : (len > cap ? (int)cap : len);
}
__device__ __forceinline__ bool bad_len(const AttnArgs &a, int b) {
    return a.lens[b] < 0 || a.lens[b] > (long long)a.table_width * PAGE;
}
// Tokens that row r (of stream b, which holds len) sees; -1 for rows past the last.
__device__ __forceinline__ int row_limit(const AttnArgs &a, int b, int len, int r) {
    if (r >= a.rows) return -1;
    return a.limits != nullptr ? max(0, min(len, a.limits[(long long)b * a.Tq + r / a.group])) : len;
}
// 2^(127 - e) for the exponent field e of a q row's largest element: finite up
// to e = 254, 0 for a row that is not (its scale is NaN).
__device__ __forceinline__ float row_inverse(int e) {
    return __uint_as_float(e == 255 ? 0u : max((uint32_t)(254 - e) << 23, 0x00400000u));  // 2^-127 is subnormal
}
// Element offset of row r of (stream b, key/value head h), for strides (sb, st, sh).
__device__ __forceinline__ long long row_at(const AttnArgs &a, int b, int h, int r, long long sb, long long st,
                                            long long sh) {
    const int t = r / a.group, g = r - t * a.group;
    return b * sb + t * st + (long long)(h * a.group + g) * sh;
}

// The dims of V in which a row that sees `limit` tokens meets a NaN code, over
// the stream's pages first, first + step, .. (count of them).  A product with
// P cannot tell: a NaN would reach the tile's other rows by way of their zeros.
// So products take such codes as numbers, and where there are any (appends
// write none) the rows that see them are looked up here.
static __device__ __noinline__ uint64_t nan_dims(const uint8_t *codes, long long page_stride, const int32_t *table,
                                                 int n_pages, int first, int step, int count, int limit) {
    uint64_t dims = 0;
    for (int i = 0, p = first; i < count && p * PAGE < limit; ++i, p += step) {
        const int id = table[p];
        if (id < 0 || id >= n_pages) continue;
        const uint32_t *w = reinterpret_cast<const uint32_t *>(codes + id * page_stride);
        const int words = min(PAGE, limit - p * PAGE) * (HD / 4);
#pragma unroll 1
        for (int j = 0; j < words; ++j) {
            const uint32_t nan = nan_codes(__ldg(w + j));
            if (nan == 0) continue;
            for (int k = 0; k < 4; ++k) dims |= (uint64_t)(nan >> (8 * k + 7) & 1) << (j % (HD / 4) * 4 + k);
        }
    }
    return dims;
}

// cache_attn_tc.cu: rows by the hundred.  Workspace bytes (0: none needed) and the launch.
size_t many_workspace(int B, int Hkv, long long rows, long long table_width);
int launch_many(const AttnArgs &a, int B, int Hkv, void *workspace, cudaStream_t stream);

}  // namespace cache
}  // namespace ress

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
// Element offset of row r of (stream b, key/value head h), for strides (sb, st, sh).
__device__ __forceinline__ long long row_at(const AttnArgs &a, int b, int h, int r, long long sb, long long st,
                                            long long sh) {
    const int t = r / a.group, g = r - t * a.group;
    return b * sb + t * st + (long long)(h * a.group + g) * sh;
}

// cache_attn_tc.cu: rows by the hundred.  Workspace bytes (0: none needed) and the launch.
size_t many_workspace(int B, int Hkv, long long rows, long long table_width);
int launch_many(const AttnArgs &a, int B, int Hkv, void *workspace, cudaStream_t stream);

}  // namespace cache
}  // namespace ress

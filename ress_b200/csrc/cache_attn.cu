// cache_attn.cu -- attention of a few queries over the paged 8-bit cache, and
// the C entry for any number (cache_attn.cuh has the definition).
#include <type_traits>

#include "cache_attn.cuh"

namespace ress {
namespace cache {

using namespace tc;

// ------------------------------------------------------------------ few rows
// Up to 16 rows a tile, on mma.sync.m16n8k16: with so few rows the bound is
// the bytes of the cache, and the 128-row tensor-core tiles would be empty.
// Each warp takes pages of its own: K and V blocks (4 KB each, K0 V0 K1 V1
// ..) arrive by bulk copies in a ring of three, so the warps never wait for
// one another before the end; sixteen warps an SM keep 64 KB or more in
// flight.  Keys (then head dims) are the MMA's 16 rows and the queries its 8
// columns, so that no half of a product is empty; the codes become fp16
// fragments in registers, once for all queries of the tile (one conversion
// per two values; e4m3 is exact in fp16):
//   S^T = K Q^T: a lane's 16-byte piece of a key row serves the four k-steps;
//      that orders the head dims differently from memory, and the q fragments
//      are loaded in the same order.
//   O^T = V^T P^T: P's 8x8 tiles are transposed in registers (movmatrix), V's
//      bytes are paired by key.  Key i of sixteen lies in row i ^ ((i >> 1) & 1),
//      so that both K's and V's shared-memory reads touch even and odd rows
//      (64-byte rows: two of equal parity meet in a bank).
// (mma.sync in e4m3 would need no conversions in the source, but measured
// slower, 142 against 122 us for 16 streams of 11 to 44 thousand tokens and 8
// heads: its operands take more instructions than these conversions.)
// The running maximum, sums and O are fp32.  q is scaled by a power of two that
// brings the row's largest element to [1, 2), and is exact in fp16 down to 2^-17
// of it (below, it errs by 2^-25 of it).  P is rounded to fp16 (2^-11), since the
// products take 16-bit operands: a page's
// probabilities count against the page's own maximum, times 2^14, so that small
// ones keep their bits; the page's weight among the others and its V scale are
// an fp32 factor of its product, so that neither costs bits.
// The pages are split over the CTAs of a cluster (and the warps of a CTA).
// Each CTA sends its rows' partial results to the shared memory of the row's
// owner, which joins them in CTA order: one launch, no workspace.  Up to 32
// streams are started longest first, so that the last CTAs are short.
// More than eight rows are two groups of the tile; what does not change from page
// to page then lies in shared memory (in registers, with the page's product
// beside O, it spilled: 16 heads x 32 queries x 43,968 tokens 52 us, 44 so).
// A NaN code among V's reaches, in the product, rows that do not see it: where
// rows see unlike parts of a page it is left out there and looked up at the end.
// 16 streams of 11 to 44 thousand tokens, 24 heads on 8: 86 us, 5.2 TB/s of the
// 6.45 that a copy reaches.  One token, 16 heads, 10,992 tokens: 11.2 us for 22.5
// MB: a launch, and three pages in turn on each warp, which is bound by the
// latency of its about 580 instructions a page (two groups: 810).
constexpr int FEW_ROWS = 16, FEW_WARPS = 8, FEW_RING = 3, FEW_SPLITS = 16;
constexpr int FEW_NT = FEW_WARPS * 32;
constexpr int FEW_SMEM = FEW_WARPS * FEW_RING * BLOCK_BYTES;
constexpr int P_SHIFT = 14;
constexpr int SLOT = HD + 4;  // floats of a partial row: O, maximum, sum
// Rows of a (stream, key/value head) up to which this kernel runs.
constexpr int FEW_MAX_ROWS = 32;

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// loads that stay where they are written
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
// Zeros in place of the NaN codes of a block in shared memory; true if there were any.
__device__ __forceinline__ bool leave_out_nans(uint32_t block, int lane) {
    bool any = false;
#pragma unroll 2
    for (int i = 0; i < 8; ++i) {
        const uint32_t at = block + (i * 32 + lane) * 16;
        uint4 u = lds128(at);
        if (!(nan_codes(u.x) | nan_codes(u.y) | nan_codes(u.z) | nan_codes(u.w))) continue;
        any = true;
        u.x &= ~((nan_codes(u.x) >> 7) * 0xFFu);
        u.y &= ~((nan_codes(u.y) >> 7) * 0xFFu);
        u.z &= ~((nan_codes(u.z) >> 7) * 0xFFu);
        u.w &= ~((nan_codes(u.w) >> 7) * 0xFFu);
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(u.x), "r"(u.y), "r"(u.z), "r"(u.w) : "memory");
    }
    any = __any_sync(0xffffffffu, any);
    if (any) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // a copy takes the block's place
        __syncwarp();
    }
    return any;
}
// shared memory of another CTA of the cluster
__device__ __forceinline__ uint32_t peer_addr(uint32_t a, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}
__device__ __forceinline__ void send4(uint32_t a, const float4 &v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(a), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
                 : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// One query row of the tile in registers: 16 head dims of lane t's, as fp16
// pairs, and the factor that turns accumulators into log2 units.
__device__ __forceinline__ float load_q16(const AttnArgs &a, int b, int h, int r, int t, uint32_t (&w)[8]) {
    float x[16] = {};
    if (r < a.rows) {
        const uint4 *p = reinterpret_cast<const uint4 *>(a.q + row_at(a, b, h, r, a.q_sb, a.q_st, a.q_sh) + t * 16);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 u = __ldg(p + i);
            const uint32_t v[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[8 * i + 2 * j] = __uint_as_float(v[j] << 16);
                x[8 * i + 2 * j + 1] = __uint_as_float(v[j] & 0xFFFF0000u);
            }
        }
    }
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) m = max(m, __float_as_uint(x[j]) & 0x7FFFFFFFu);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const int e = (int)(m >> 23);
    const float inv = row_inverse(e);
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = half2_bits(x[2 * j] * inv, x[2 * j + 1] * inv);
    return scale_value(e) * a.scale_log2;
}

// The stream that CTAs of index z work on: the z-th longest of up to 32.
__device__ __forceinline__ int stream_by_length(const AttnArgs &a, int z, int streams) {
    if (streams == 1 || streams > 32) return z;
    const int lane = threadIdx.x & 31, len = lane < streams ? a.lens[lane] : INT_MIN;
    int rank = 0;
    for (int j = 0; j < streams; ++j) {
        const int other = __shfl_sync(0xffffffffu, len, j);
        rank += other > len || (other == len && j < lane);
    }
    return __ffs(__ballot_sync(0xffffffffu, lane < streams && rank == z)) - 1;
}

// NT: groups of eight rows in the tile.
template <int NT>
__global__ void __launch_bounds__(FEW_NT, 2) few_kernel(const AttnArgs a, int kv_heads) {
    extern __shared__ __align__(128) unsigned char dyn[];
    __shared__ uint64_t full[FEW_WARPS][FEW_RING];
    __shared__ int abort_s;
    __shared__ float part_m[FEW_WARPS][FEW_ROWS], part_l[FEW_WARPS][FEW_ROWS];
    // what the cluster's CTAs send to this one: for its n-th row, one slot per CTA
    __shared__ __align__(16) float inbox[FEW_ROWS * SLOT + FEW_SPLITS * SLOT];
    const int split = blockIdx.x, splits = gridDim.x;
    const int h = blockIdx.y % kv_heads, tile = blockIdx.y / kv_heads, b = stream_by_length(a, blockIdx.z, gridDim.z);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int r0 = tile * FEW_ROWS, rows = min(FEW_ROWS, a.rows - r0);
    volatile int *abort_flag = &abort_s;
    if (threadIdx.x < FEW_WARPS * FEW_RING) mbar_init(&full[0][0] + threadIdx.x, 1);
    if (threadIdx.x == 0) abort_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    // what the rows see; a lane works on rows 2t and 2t + 1 of each group
    const int len = stream_len(a, b);
    int lim[NT][2], lo = len, hi = len;
    if (a.limits != nullptr) {
        lo = INT_MAX;
        hi = 0;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                lim[n][e] = row_limit(a, b, len, r0 + 8 * n + 2 * t + e);
                if (lim[n][e] >= 0) {
                    lo = min(lo, lim[n][e]);
                    hi = max(hi, lim[n][e]);
                }
            }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (a.limits == nullptr || lim[n][e] < 0) lim[n][e] = hi;  // rows past the last: computed, never written
    __syncthreads();
    // they have started; waited for before the first store into a peer
    if (splits > 1) cluster_arrive_relaxed();
    if (threadIdx.x == 0 && split == 0 && bad_len(a, b)) atomicOr(a.status, RESS_STATUS_CACHE_RANGE);

    // this warp's pages: first, first + FEW_WARPS, ... (count of them)
    const int pages = (hi + PAGE - 1) / PAGE;
    const int p0 = (int)((long long)pages * split / splits), p1 = (int)((long long)pages * (split + 1) / splits);
    const int first = p0 + warp, count = p1 > first ? (p1 - first + FEW_WARPS - 1) / FEW_WARPS : 0;
    // page ids and scales, 32 pages at a time: lane i holds page base + i
    const int32_t *table = a.table + b * a.table_stride;
    auto fetch_id = [&](int base) {
        const int i = base + lane;
        int id = i < count ? table[first + i * FEW_WARPS] : 0;
        if (id < 0 || id >= a.n_pages) {  // no such page: its tokens count as NaN
            atomicOr(a.status, RESS_STATUS_CACHE_RANGE);
            id = -1;
        }
        return id;
    };
    auto fetch_scale = [&](const Pages &P, int id) { return id < 0 ? 255 : (int)P.scale[id * P.scale_stride + h]; };
    int id_a = fetch_id(0), id_b = 0;  // batches of even and odd number
    unsigned char *ring = dyn + warp * FEW_RING * BLOCK_BYTES;
    const uint32_t ring_a = smem_u32(ring);
    const int blocks = 2 * count;
    int fill_slot = 0;  // ring slot of the next block to ask for
    auto issue = [&](int n) {  // block n: K (even) or V of page n / 2; all lanes call it
        const int i = n >> 1, id = max(__shfl_sync(0xffffffffu, (i & 32) ? id_b : id_a, i & 31), 0);
        if (lane == 0) {
            const Pages &P = n & 1 ? a.V : a.K;
            mbar_expect_tx(&full[warp][fill_slot], BLOCK_BYTES);
            bulk_load(ring_a + fill_slot * BLOCK_BYTES, P.codes + id * P.page_stride + h * P.head_stride, BLOCK_BYTES,
                      &full[warp][fill_slot]);
        }
        if (++fill_slot == FEW_RING) fill_slot = 0;
    };
    int issued = 0;
    while (issued < min(blocks, FEW_RING)) issue(issued++);
    // the scales, behind the first copies
    int uk_a = fetch_scale(a.K, id_a), uv_a = fetch_scale(a.V, id_a), uk_b = 0, uv_b = 0;
    if (count > 32) {
        id_b = fetch_id(32);
        uk_b = fetch_scale(a.K, id_b);
        uv_b = fetch_scale(a.V, id_b);
    }

    uint32_t q[NT][8];
    float rf[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const float f = load_q16(a, b, h, r0 + 8 * n + g, t, q[n]);
        rf[n][0] = __shfl_sync(0xffffffffu, f, 8 * t);  // of row 2t: its lanes are 4 * 2t ..
        rf[n][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
    }
    // Two groups leave no registers for what does not change: it is read again for every page.
    __shared__ __align__(16) uint32_t q_s[4][32][4];
    __shared__ __align__(8) int lim_s[FEW_ROWS];
    __shared__ __align__(8) float rf_s[FEW_ROWS];
    if constexpr (NT == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t *w = &q[i >> 1][4 * (i & 1)];
            if (warp == i) *reinterpret_cast<uint4 *>(q_s[i][lane]) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        if (warp == 0 && g == 0) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    lim_s[8 * n + 2 * t + e] = lim[n][e];
                    rf_s[8 * n + 2 * t + e] = rf[n][e];
                }
        }
        __syncthreads();
    }

    bool nan_seen = false;  // a page's NaN codes were left out
    float o[NT][4][4] = {};
    float m[NT][2], l[NT][2] = {};  // sums count in 2^-P_SHIFT
    const float down = scale_value(127 - P_SHIFT);
#pragma unroll
    for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = -INFINITY;
    const int pg = g ^ ((g >> 1) & 1);  // this lane's key of eight in S^T
    const int kf = 2 * t + (t & 1), kh = 2 * t + 1 - (t & 1);  // and its pair of keys in V^T
    const uint32_t koff = (uint32_t)pg * HD + t * 16;
    int slot = 0, phase = 0;  // of the block consumed next
    auto take = [&]() -> const unsigned char * {
        if (!wait_bar_warp(&full[warp][slot], phase, abort_flag, a.status)) return nullptr;
        return ring + slot * BLOCK_BYTES;
    };
    auto done = [&]() {  // the block taken last is in registers: its slot takes the next one
        __syncwarp();
        if (issued < blocks) issue(issued++);
        if (++slot == FEW_RING) {
            slot = 0;
            phase ^= 1;
        }
    };
    for (int i = 0; i < count; ++i) {
        // the batch two ahead replaces the one just used up
        if ((i & 31) == 0 && i > 0 && i + 32 < count) {
            if (i & 32) {
                id_a = fetch_id(i + 32);
                uk_a = fetch_scale(a.K, id_a);
                uv_a = fetch_scale(a.V, id_a);
            } else {
                id_b = fetch_id(i + 32);
                uk_b = fetch_scale(a.K, id_b);
                uv_b = fetch_scale(a.V, id_b);
            }
        }
        const int uk = __shfl_sync(0xffffffffu, (i & 32) ? uk_b : uk_a, i & 31);
        const int uv = __shfl_sync(0xffffffffu, (i & 32) ? uv_b : uv_a, i & 31);
        const unsigned char *sk = take();
        if (sk == nullptr) break;
        if constexpr (NT == 2) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint4 u = lds128(smem_u32(q_s[j][lane]));
                uint32_t *w = &q[j >> 1][4 * (j & 1)];
                w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
            }
        }
        float c[4][NT][4] = {};  // sixteen keys each: keys pg (0, 1) and pg + 8 (2, 3) of rows 2t, 2t + 1
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
            const uint4 ka = lds128(smem_u32(sk) + mt * 16 * HD + koff), kb = lds128(smem_u32(sk) + (mt * 16 + 8) * HD + koff);
#pragma unroll
            for (int st = 0; st < 4; ++st) {
                const uint32_t x = st == 0 ? ka.x : st == 1 ? ka.y : st == 2 ? ka.z : ka.w;
                const uint32_t y = st == 0 ? kb.x : st == 1 ? kb.y : st == 2 ? kb.z : kb.w;
                const uint32_t a0 = e4m3_to_half2((uint16_t)x), a1 = e4m3_to_half2((uint16_t)y);
                const uint32_t a2 = e4m3_to_half2((uint16_t)(x >> 16)), a3 = e4m3_to_half2((uint16_t)(y >> 16));
#pragma unroll
                for (int n = 0; n < NT; ++n) mma_16816(c[mt][n], a0, a1, a2, a3, q[n][2 * st], q[n][2 * st + 1]);
            }
        }
        done();
        const int base = (first + i * FEW_WARPS) * PAGE;
        const float fk = scale_value(uk), fv = scale_value(uv) * down;
        // where every row sees the whole page there are no masks (a tenth of the instructions)
        auto page = [&](auto page_whole) {
            constexpr bool whole = decltype(page_whole)::value;
            if constexpr (NT == 2) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint2 u = lds64(smem_u32(&rf_s[8 * n + 2 * t]));
                    rf[n][0] = __uint_as_float(u.x);
                    rf[n][1] = __uint_as_float(u.y);
                    if (!whole) {
                        const uint2 w = lds64(smem_u32(&lim_s[8 * n + 2 * t]));
                        lim[n][0] = (int)w.x;
                        lim[n][1] = (int)w.y;
                    }
                }
            }
            uint32_t pb[NT][4][2];
            float f[NT][2];  // of the page's product
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float bias[2], cs[2], alpha[2], sum[2] = {};
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = -INFINITY;
#pragma unroll
                    for (int mt = 0; mt < 4; ++mt) {
                        if (!whole) {  // hidden tokens: -inf, whatever lies there
                            if (base + mt * 16 + pg >= lim[n][e]) c[mt][n][e] = -INFINITY;
                            if (base + mt * 16 + 8 + pg >= lim[n][e]) c[mt][n][e + 2] = -INFINITY;
                        }
                        top = fmaxf(top, fmaxf(c[mt][n][e], c[mt][n][e + 2]));
                    }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    cs[e] = rf[n][e] * fk;  // not negative; a NaN one shows in the exponentials
                    top = top == -INFINITY ? top : top * cs[e];
                    bias[e] = P_SHIFT - (top == -INFINITY ? 0.0f : top);
                    const float mn = fmaxf(m[n][e], top);
                    const float mb = mn == -INFINITY ? 0.0f : mn;
                    alpha[e] = ex2(m[n][e] - mb);
                    f[n][e] = ex2(top - mb);
                    m[n][e] = mn;
                }
                if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        o[n][d][0] *= alpha[0];
                        o[n][d][1] *= alpha[1];
                        o[n][d][2] *= alpha[0];
                        o[n][d][3] *= alpha[1];
                    }
                }
                // P: probabilities for the sums, and times the V scale as fp16 fragments
#pragma unroll
                for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float p[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            p[e] = ex2(fmaf(c[mt][n][2 * k + e], cs[e], bias[e]));
                            // a hidden token is 0 even where a factor is 0 or NaN
                            if (!whole && base + mt * 16 + 8 * k + pg >= lim[n][e]) p[e] = 0.0f;
                            sum[e] += p[e];
                        }
                        pb[n][mt][k] = transpose8x8(half2_bits(p[0], p[1]));
                    }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    l[n][e] = fmaf(sum[e], f[n][e], l[n][e] * alpha[e]);
                    // a row that sees none of the page takes nothing from it, a NaN scale neither
                    f[n][e] = whole || base < lim[n][e] ? f[n][e] * fv : 0.0f;
                }
            }
            const unsigned char *sv = take();
            if (sv == nullptr) return false;
            // where rows see unlike parts of the page
            if (!whole && lo != hi && leave_out_nans(smem_u32(sv), lane)) nan_seen = true;
            float x[NT][4][4] = {};  // the page's product
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
                const uint32_t va = smem_u32(sv) + mt * 16 * HD + g * 8;
                uint2 v0 = lds64(va + kf * HD), v1 = lds64(va + kh * HD);
                uint2 v2 = lds64(va + (8 + kf) * HD), v3 = lds64(va + (8 + kh) * HD);
                if (!whole && base + PAGE > hi) {  // slots that no row sees hold anything, NaN codes too
                    const int e = hi - base - 16 * mt;
                    if (kf >= e) v0 = make_uint2(0, 0);
                    if (kh >= e) v1 = make_uint2(0, 0);
                    if (8 + kf >= e) v2 = make_uint2(0, 0);
                    if (8 + kh >= e) v3 = make_uint2(0, 0);
                }
#pragma unroll
                for (int d = 0; d < 4; d += 2) {  // dims 8g + d, and + 4 in the lower half of the rows
                    const uint32_t sel = d == 0 ? 0x5140u : 0x7362u;
                    const uint32_t y0 = __byte_perm(v0.x, v1.x, sel), y1 = __byte_perm(v0.y, v1.y, sel);
                    const uint32_t y2 = __byte_perm(v2.x, v3.x, sel), y3 = __byte_perm(v2.y, v3.y, sel);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint32_t a0 = e4m3_to_half2((uint16_t)(y0 >> (16 * k))), a1 = e4m3_to_half2((uint16_t)(y1 >> (16 * k)));
                        const uint32_t a2 = e4m3_to_half2((uint16_t)(y2 >> (16 * k))), a3 = e4m3_to_half2((uint16_t)(y3 >> (16 * k)));
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma_16816(x[n][d + k], a0, a1, a2, a3, pb[n][mt][0], pb[n][mt][1]);
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int j = 0; j < 4; j += 2) {
                        const f32x2 y = f2_fma_rn(f2_pack(x[n][d][j], x[n][d][j + 1]), f2_pack(f[n][0], f[n][1]),
                                                  f2_pack(o[n][d][j], o[n][d][j + 1]));
                        f2_unpack(y, o[n][d][j], o[n][d][j + 1]);
                    }
            return true;
        };
        if (!(base + PAGE <= lo ? page(std::true_type{}) : page(std::false_type{}))) break;
        done();
    }
    // copies in flight land before their ring is used again (all have, unless a wait ran out)
    for (int s = 0; s < min(issued, FEW_RING); ++s) {
        const int last = issued - 1 - ((issued - 1 - s) % FEW_RING);
        const uint64_t t0 = globaltimer();
        while (!mbar_try_wait(smem_u32(&full[warp][s]), (last / FEW_RING) & 1) && globaltimer() - t0 < TIMEOUT_NS) {
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int d = 4; d < 32; d *= 2) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
            if (g == 0) {
                part_m[warp][8 * n + 2 * t + e] = m[n][e];
                part_l[warp][8 * n + 2 * t + e] = l[n][e] * down;
            }
        }
    __syncthreads();
    // the warps' O meet in the ring, 4 KB a warp
    float *po = reinterpret_cast<float *>(dyn) + warp * FEW_ROWS * HD;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int k = 0; k < 2; ++k)
                *reinterpret_cast<float4 *>(po + (8 * n + 2 * t + e) * HD + 8 * g + 4 * k) =
                    make_float4(o[n][0][e + 2 * k], o[n][1][e + 2 * k], o[n][2][e + 2 * k], o[n][3][e + 2 * k]);
    if (nan_seen) {
        __syncwarp();
        const uint64_t dims = nan_dims(a.V.codes + h * a.V.head_stride, a.V.page_stride, table, a.n_pages, first, FEW_WARPS,
                                       count, lane < 8 * NT ? row_limit(a, b, len, r0 + lane) : 0);
        for (int d = 0; d < HD; ++d)
            if (dims >> d & 1) po[lane * HD + d] = NAN;
    }
    __syncthreads();
    if (splits > 1) cluster_wait();  // the peers have started
    const float *co = reinterpret_cast<const float *>(dyn);
    auto write = [&](int r, int d, float4 acc, float l) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no token seen: zeros
        const long long at = row_at(a, b, h, r0 + r, a.o_sb, a.o_st, a.o_sh) + d;
        if (a.out_bf16) {
            const __nv_bfloat162 x = __floats2bfloat162_rn(acc.x * inv, acc.y * inv);
            const __nv_bfloat162 y = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
            *reinterpret_cast<uint2 *>(reinterpret_cast<__nv_bfloat16 *>(a.out) + at) =
                make_uint2(*reinterpret_cast<const uint32_t *>(&x), *reinterpret_cast<const uint32_t *>(&y));
        } else {
            *reinterpret_cast<float4 *>(reinterpret_cast<float *>(a.out) + at) =
                make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
        }
    };
    if (threadIdx.x < rows * 16) {
        const int r = threadIdx.x >> 4, d = (threadIdx.x & 15) * 4;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < FEW_WARPS; ++w) mm = fmaxf(mm, part_m[w][r]);
        const float mb = mm == -INFINITY ? 0.0f : mm;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.0f;
#pragma unroll
        for (int w = 0; w < FEW_WARPS; ++w) {
            const float f = ex2(part_m[w][r] - mb);
            const float4 v = *reinterpret_cast<const float4 *>(co + (w * FEW_ROWS + r) * HD + d);
            acc.x += f * v.x;
            acc.y += f * v.y;
            acc.z += f * v.z;
            acc.w += f * v.w;
            l += f * part_l[w][r];
        }
        if (splits == 1) {
            write(r, d, acc, l);
        } else {
            // row r goes to CTA r % splits, as its (r / splits)-th row
            const uint32_t to = smem_u32(inbox) + (uint32_t)((r / splits) * splits + split) * SLOT * 4;
            send4(peer_addr(to + d * 4, r % splits), acc);
            if (d == 0) send4(peer_addr(to + HD * 4, r % splits), make_float4(mm, l, 0.f, 0.f));
        }
    }
    if (splits == 1) return;
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    const int mine = threadIdx.x >> 4, d = (threadIdx.x & 15) * 4, r = mine * splits + split;
    if (r < rows) {
        const float *in = inbox + mine * splits * SLOT;
        float mm = -INFINITY;
        for (int s = 0; s < splits; ++s) mm = fmaxf(mm, in[s * SLOT + HD]);
        const float mb = mm == -INFINITY ? 0.0f : mm;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.0f;
        for (int s = 0; s < splits; ++s) {
            const float f = ex2(in[s * SLOT + HD] - mb);
            const float4 v = *reinterpret_cast<const float4 *>(in + s * SLOT + d);
            acc.x += f * v.x;
            acc.y += f * v.y;
            acc.z += f * v.z;
            acc.w += f * v.w;
            l += f * in[s * SLOT + HD + 1];
        }
        write(r, d, acc, l);
    }
}

// Clusters of more than eight CTAs, once per device and kernel.
static bool allow_wide_clusters(const void *kern, int which) {
    static thread_local uint64_t done[2] = {0, 0};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 64 && (done[which] >> dev) & 1) return true;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return false;
    if (dev < 64) done[which] |= 1ull << dev;
    return true;
}

static int launch_few(const AttnArgs &a, int B, int Hkv, cudaStream_t stream) {
    const int tiles = (a.rows + FEW_ROWS - 1) / FEW_ROWS;
    if ((long long)tiles * Hkv > 65535) return RESS_E_SHAPE;  // the grid's second dimension
    const long long groups = (long long)tiles * Hkv * B;
    // CTAs per (rows, head, stream).  While the CTAs fit on an SM each, pages enough
    // for half a CTA's warps suffice (1 x 16 heads x 1,374 tokens: 9.6 us in one
    // CTA, 6.5 in four, 6.7 in eight); beyond that two pages a warp, and CTAs
    // for four per SM, so that the longer streams' can start first (16 x 8 heads
    // x 11 to 44 thousand: 122 us in two, 113 in four, 118 in eight).  Sixteen
    // CTAs make a cluster that is hard to place: only where eight leave half of
    // the GPU idle.  (CTAs of sixteen warps, one an SM, gain nothing: one token,
    // 16 heads x 10,992: 12.3 us in four of them, 12.2 in eight of eight warps,
    // and 17.1 in eight, which are not all placed at once.)
    int splits = 1;
    const long long width = a.table_width;
    while (splits < 8 && groups * splits * 2 <= 148 && splits * 2 * FEW_WARPS / 2 <= width) splits *= 2;
    while (splits < 8 && groups * splits * 2 <= 148 * 4 && splits * 2 * FEW_WARPS * 2 <= width) splits *= 2;
    if (splits == 8 && groups * 16 <= 148 && 16 * FEW_WARPS <= width) splits = 16;
    auto kern = a.rows <= 8 ? few_kernel<1> : few_kernel<2>;
    set_smem_attr((const void *)kern, FEW_SMEM);
    if (splits > 8 && !allow_wide_clusters((const void *)kern, a.rows <= 8)) return RESS_E_LAUNCH;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(splits, (unsigned)(tiles * Hkv), (unsigned)B);
    cfg.blockDim = dim3(FEW_NT);
    cfg.dynamicSmemBytes = FEW_SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = splits;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, a, Hkv) == cudaSuccess ? RESS_OK : RESS_E_LAUNCH;
}

}  // namespace cache
}  // namespace ress

using namespace ress;

extern "C" size_t ress_cache_attn_workspace(int64_t streams, int64_t heads, int64_t rows, int64_t table_width) {
    if (streams <= 0 || heads <= 0 || rows <= cache::FEW_MAX_ROWS || table_width <= 0) return 0;
    return cache::many_workspace((int)streams, (int)heads, rows, table_width);
}

extern "C" int ress_cache_attn(const ress_cache *cache, const ress_attn_args *args, int32_t *status,
                               ress_stream_t stream) {
    const int rc = cache::check_cache(cache);
    if (rc != RESS_OK) return rc;
    if (!args || !status || !args->q || !args->out || args->tokens <= 0) return RESS_E_ARG;
    const ress_attn_args &g = *args;
    const int64_t H = cache->heads;
    if (g.q_heads <= 0 || g.q_heads % H != 0 || !(g.sm_scale >= 0)) return RESS_E_ARG;
    if (((uintptr_t)g.q & 15) || ((g.q_sb | g.q_st | g.q_sh) & 7)) return RESS_E_ARG;
    const int size = g.out_bf16 ? 2 : 4;
    if (((uintptr_t)g.out & 15) || (((g.o_sb | g.o_st | g.o_sh) * size) & 15)) return RESS_E_ARG;
    if (g.tokens > (1 << 30) || g.q_heads > (1 << 20)) return RESS_E_SHAPE;
    const int64_t rows = g.tokens * (g.q_heads / H);
    if (rows > (1 << 30)) return RESS_E_SHAPE;
    cache::AttnArgs a;
    a.q = g.q;
    a.q_sb = g.q_sb; a.q_st = g.q_st; a.q_sh = g.q_sh;
    a.out = g.out;
    a.o_sb = g.o_sb; a.o_st = g.o_st; a.o_sh = g.o_sh;
    a.out_bf16 = g.out_bf16 != 0;
    a.Tq = (int)g.tokens;
    a.group = (int)(g.q_heads / H);
    a.rows = (int)rows;
    a.K = {cache->k_pages, cache->k_scale, cache->page_stride, cache->head_stride, cache->scale_stride};
    a.V = {cache->v_pages, cache->v_scale, cache->page_stride, cache->head_stride, cache->scale_stride};
    a.table = cache->table; a.lens = cache->lens; a.limits = g.limits;
    a.table_stride = cache->table_stride; a.table_width = (int)cache->table_width; a.n_pages = (int)cache->n_pages;
    a.scale_log2 = (float)(g.sm_scale * 1.4426950408889634);
    a.status = status;
    a.partial = nullptr;
    a.arrived = nullptr;
    if (rows > cache::FEW_MAX_ROWS)
        return cache::launch_many(a, (int)cache->streams, (int)H, args->workspace, (cudaStream_t)stream);
    return cache::launch_few(a, (int)cache->streams, (int)H, (cudaStream_t)stream);
}

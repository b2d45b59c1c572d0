// cache_attn_tc.cu -- attention of many queries over the paged 8-bit cache on
// the tensor cores (cache_attn.cuh has the definition).
//
// One CTA per 256 rows of a (stream, key/value head), as two tiles of 128
// that share every page of keys and values; 24 warps:
//   warp 0       loads pages: K blocks (TMA, 64B-swizzled), V blocks (bulk);
//   warp 1       issues S = Q K^T, tcgen05.mma kind::f8f6f4.  K's codes are an
//                operand as they lie in the cache.  q is split into two e4m3
//                parts, q = hi + lo (4 + 4 significant bits, as many as bf16
//                has), so S takes four K = 32 steps: hi and lo against the same
//                K, which is what bf16 would take.  Scales are applied to S.
//   warp 2       issues O += P V, kind::f16 in bf16.  N = 80: sixteen columns
//                of ones give the row sums of P.
//   warp 3       allocates tensor memory.
//   warps 4-7    turn V's codes into bf16 (exact: the scale is a power of two)
//                in the 128B-swizzled layout that the MMA reads, once for both
//                tiles.
//   warps 8-23   softmax, eight warps a tile, two threads per row: thread =
//                (row, 32 of the page's 64 keys).  The running maximum moves
//                only when it grows by more than 2^8, so O in tensor memory is
//                rarely rescaled.
// Pages that all rows of a tile see take the hot path; the first page and
// those that a limit cuts run out of line.  P is rounded to bf16 for the MMA,
// numerator and denominator alike; everything else is fp32.
// When the tiles are too few for the GPU the pages are split over several
// CTAs; the one that finishes last joins the pieces in page order, so the
// result does not depend on the order of arrival.
// Every wait is bounded (tcgen05.cuh).  No TMA multicast.
#include "cache_attn.cuh"

namespace ress {
namespace cache {
namespace many {

using namespace tc;

constexpr int NT = 768, TILE = 128, TILES = 2, NSOFT = 256;  // softmax threads of a tile
constexpr int NK = 6, NC = 6, NV = 3, NP = 3;                // rings: K, V codes, V in bf16, P
constexpr int INFO = 32;  // scales of pages in flight: more than any ring is deep
constexpr int REGS_CTRL = 32, REGS_SOFT = 104;
static_assert(256 * REGS_CTRL + 512 * REGS_SOFT <= NT * 80, "register split above the launch's registers");
constexpr int Q_BYTES = TILE * 128, V_BYTES = PAGE * 128, P_BYTES = TILE * 128, ONES_BYTES = 16 * 128;
constexpr int OFF_Q = 0;
constexpr int OFF_K = OFF_Q + TILES * Q_BYTES;
constexpr int OFF_C = OFF_K + NK * BLOCK_BYTES;
constexpr int OFF_V = OFF_C + NC * BLOCK_BYTES;
constexpr int OFF_P = OFF_V + NV * V_BYTES;
constexpr int OFF_ONES = OFF_P + TILES * NP * P_BYTES;
constexpr int SMEM = OFF_ONES + ONES_BYTES + 1024;
static_assert(V_BYTES == 4 * 2048, "four K = 16 slices a page");
static_assert(SMEM + 4096 <= 227 * 1024, "shared memory");
constexpr float RESCALE_THRESH = 8.0f;
constexpr int SPLIT_MAX = 8, PART_ROW = HD + 4;  // a partial row: O, maximum, sum

// D f32; A, B e4m3, K-major; N = 64.  And D f32; A, B bf16, B MN-major; N = 80.
constexpr uint32_t IDESC_S = (1u << 4) | ((64u >> 3) << 17) | ((128u >> 4) << 24);
constexpr uint32_t IDESC_O =
    (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((80u >> 3) << 17) | ((128u >> 4) << 24);

struct Bars {
    uint64_t k_full[NK], k_empty[NK], c_full[NC], c_empty[NC], v_full[NV], v_empty[NV];
    uint64_t s_full[TILES][2], s_free[TILES][2], p_full[TILES][NP], o_full[TILES][NP];
    uint64_t s_done, pv_done;
    uint32_t tmem;
    int abort_flag, hi, lo[TILES], join[TILES];
    int info[INFO];
    int lim[TILES * TILE];
    float unit[TILES * TILE];  // of a row's S, in log2 units, K's scale aside
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, uint64_t *bar, int x, int y, int z,
                                            int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::
            "r"(dst),
        "l"((uint64_t)map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void mma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(IDESC_S), "r"(acc));
}
// One lane of a converged warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// Four e4m3 codes to bf16 pairs (0, 2) and (1, 3).  A code's exponent and
// significand bits, moved into a bf16's place, are its value times 2^-120
// (the biases are 7 and 127; subnormals as well): one multiplication by
// 2^120 and the page's scale is exact.
__device__ __forceinline__ void codes_to_bf16(uint32_t w, uint32_t f, uint32_t &even, uint32_t &odd) {
    even = mul_bf16x2(((w << 8) & 0x80008000u) | ((w & 0x007F007Fu) << 4), f);
    odd = mul_bf16x2((w & 0x80008000u) | ((w & 0x7F007F00u) >> 4), f);
}
// 2^e as a bf16 pair
__device__ __forceinline__ uint32_t pow2_bf16x2(int e) { return (uint32_t)((e + 127) << 7) * 0x00010001u; }

// What an out-of-line softmax step needs of its thread.
struct Row {
    uint32_t tS, tO, lane_addr, sP, prow, rsw, ch0;
    int col0;
    uint64_t *o_full, *s_free;
    volatile int *abort_flag;
    int32_t *status;
};

// This thread's half of its row of O (and of the row-sum columns) times alpha.
__device__ __noinline__ void rescale_o(uint32_t tO, uint32_t lane_addr, float alpha) {
    uint32_t o[32], s8[8];
    tmem_ld_half32(tO + lane_addr, o);
    tmem_ld_half8(tO + HD + lane_addr, s8);
    tmem_wait_ld();
#pragma unroll
    for (int t = 0; t < 32; ++t) o[t] = __float_as_uint(__uint_as_float(o[t]) * alpha);
#pragma unroll
    for (int t = 0; t < 8; ++t) s8[t] = __float_as_uint(__uint_as_float(s8[t]) * alpha);
    tmem_st_half32(tO + lane_addr, o);
    tmem_st_half8(tO + HD + lane_addr, s8);
    tmem_wait_st();
}

// The general step for page j: the row sees the page's first `seen` keys, its
// maximum may not be set yet.  Returns the new maximum, NaN when a wait failed.
__device__ __noinline__ float step_general(const Row &rc, int j, int seen, float c, float m) {
    const int sb = j & 1, pb = j % NP;
    uint32_t sv[32];
    tmem_ld_half32(rc.tS + sb * 64 + rc.lane_addr, sv);
    tmem_wait_ld();
    fence_before();
    mbar_arrive(rc.s_free + sb);
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < 32; ++t) {
        const float x = rc.col0 + t < seen ? __uint_as_float(sv[t]) * c : -INFINITY;
        sv[t] = __float_as_uint(x);
        mx = fmaxf(mx, x);
    }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));  // the row's other half
    const bool grow = mx > m + RESCALE_THRESH;             // m = -inf: whenever a key is seen
    const float m_new = grow ? mx : m;
    if (__any_sync(0xffffffffu, grow && j > 0)) {
        const int pj = j - 1;
        if (!wait_bar_warp(rc.o_full + pj % NP, (pj / NP) & 1, rc.abort_flag, rc.status))
            return __int_as_float(0x7fffffff);
        fence_after();
        rescale_o(rc.tO, rc.lane_addr, grow ? ex2(m - m_new) : 1.0f);
    }
    const float mb = m_new == -INFINITY ? 0.0f : m_new;
#pragma unroll
    for (int ch = 0; ch < 4; ++ch) {
        uint32_t h[4];
#pragma unroll
        for (int t = 0; t < 8; t += 2)
            h[t >> 1] = pack_bf16(ex2(__uint_as_float(sv[ch * 8 + t]) - mb), ex2(__uint_as_float(sv[ch * 8 + t + 1]) - mb));
        sts128(rc.sP + pb * P_BYTES + rc.prow + (((rc.ch0 + (uint32_t)ch) ^ rc.rsw) << 4), h[0], h[1], h[2], h[3]);
    }
    fence_before();
    return m_new;
}

// Half a row (32 dims from col0) to the output, times inv.
__device__ __forceinline__ void store_row(const AttnArgs &a, long long at, const float (&o)[32], float inv) {
    if (a.out_bf16) {
        uint4 *p = reinterpret_cast<uint4 *>(reinterpret_cast<__nv_bfloat16 *>(a.out) + at);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            p[i] = make_uint4(pack_bf16(o[8 * i] * inv, o[8 * i + 1] * inv), pack_bf16(o[8 * i + 2] * inv, o[8 * i + 3] * inv),
                              pack_bf16(o[8 * i + 4] * inv, o[8 * i + 5] * inv),
                              pack_bf16(o[8 * i + 6] * inv, o[8 * i + 7] * inv));
    } else {
        float4 *p = reinterpret_cast<float4 *>(reinterpret_cast<float *>(a.out) + at);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            p[i] = make_float4(o[4 * i] * inv, o[4 * i + 1] * inv, o[4 * i + 2] * inv, o[4 * i + 3] * inv);
    }
}

__global__ void __launch_bounds__(NT, 1)
    many_kernel(const __grid_constant__ CUtensorMap tm_k, const AttnArgs a, int row_ctas, int splits) {
    extern __shared__ unsigned char raw[];
    __shared__ Bars B;
    unsigned char *smem = reinterpret_cast<unsigned char *>(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    const uint32_t sQ = smem_u32(smem + OFF_Q), sK = smem_u32(smem + OFF_K), sC = smem_u32(smem + OFF_C);
    const uint32_t sV = smem_u32(smem + OFF_V), sOnes = smem_u32(smem + OFF_ONES);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int cta = blockIdx.x % row_ctas, split = blockIdx.x / row_ctas, h = blockIdx.y, b = blockIdx.z;
    const int r0 = cta * TILE * TILES;
    const int nt = a.rows - r0 > TILE ? 2 : 1;  // tiles with rows
    volatile int *abort_flag = &B.abort_flag;
    const int len = stream_len(a, b);

    if (tid == 0) {
        for (int i = 0; i < NK; ++i) {
            mbar_init(&B.k_full[i], 1);
            mbar_init(&B.k_empty[i], 1);
        }
        for (int i = 0; i < NC; ++i) {
            mbar_init(&B.c_full[i], 1);
            mbar_init(&B.c_empty[i], 128);
        }
        for (int i = 0; i < NV; ++i) {
            mbar_init(&B.v_full[i], 128);
            mbar_init(&B.v_empty[i], 1);
        }
        for (int t = 0; t < TILES; ++t) {
            for (int i = 0; i < 2; ++i) {
                mbar_init(&B.s_full[t][i], 1);
                mbar_init(&B.s_free[t][i], NSOFT);
            }
            for (int i = 0; i < NP; ++i) {
                mbar_init(&B.p_full[t][i], NSOFT);
                mbar_init(&B.o_full[t][i], 1);
            }
            B.lo[t] = INT_MAX;
        }
        mbar_init(&B.s_done, 1);
        mbar_init(&B.pv_done, 1);
        B.abort_flag = 0;
        B.hi = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (split == 0 && bad_len(a, b)) atomicOr(a.status, RESS_STATUS_CACHE_RANGE);
    }
    if (warp == 3) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&B.tmem)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    __syncthreads();
    if (tid < ONES_BYTES / 16) sts128(sOnes + tid * 16, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u);
    if (tid < TILES * TILE) {
        const int l = row_limit(a, b, len, r0 + tid);
        B.lim[tid] = l;
        if (l >= 0) {
            atomicMax(&B.hi, l);
            atomicMin(&B.lo[tid / TILE], l);
        }
    } else {
        // q of one row, 32 dims a thread: scaled by a power of two to [128, 256), split into two e4m3 parts
        const int i = tid - TILES * TILE, row = i >> 1, half = i & 1;
        uint4 u[4] = {};
        if (r0 + row < a.rows) {
            const uint4 *p = reinterpret_cast<const uint4 *>(a.q + row_at(a, b, h, r0 + row, a.q_sb, a.q_st, a.q_sh) + half * 32);
#pragma unroll
            for (int k = 0; k < 4; ++k) u[k] = __ldg(p + k);
        }
        uint32_t am = 0;
        const uint32_t *w = reinterpret_cast<const uint32_t *>(u);
#pragma unroll
        for (int k = 0; k < 16; ++k) am = max(am, max((w[k] << 16) & 0x7FFFFFFFu, w[k] & 0x7FFF0000u));
        am = max(am, __shfl_xor_sync(0xffffffffu, am, 1));
        const int e = max((int)(am >> 23), 8);  // 2^(134 - e) stays in range, for a zero row as well
        const float f = scale_inverse(e) * 128.0f;
        const uint32_t base = sQ + (row / TILE) * Q_BYTES + (row % TILE) * 128;
#pragma unroll
        for (int k = 0; k < 2; ++k) {  // 16 dims: one 16-byte piece of each part
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                float x[4], y[4];
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const uint32_t ww = w[k * 8 + n * 2 + v];
                    x[2 * v] = __uint_as_float(ww << 16) * f;
                    x[2 * v + 1] = __uint_as_float(ww & 0xFFFF0000u) * f;
                }
                hi[n] = e4m3x4(x[0], x[1], x[2], x[3]);
                const uint32_t h01 = e4m3_to_half2((uint16_t)hi[n]), h23 = e4m3_to_half2((uint16_t)(hi[n] >> 16));
                const float2 f01 = __half22float2(*reinterpret_cast<const __half2 *>(&h01));
                const float2 f23 = __half22float2(*reinterpret_cast<const __half2 *>(&h23));
                y[0] = x[0] - f01.x;
                y[1] = x[1] - f01.y;
                y[2] = x[2] - f23.x;
                y[3] = x[3] - f23.y;
                lo[n] = e4m3x4(y[0], y[1], y[2], y[3]);
            }
            const uint32_t sw = (uint32_t)(row & 7);
            sts128(base + (((uint32_t)(half * 2 + k) ^ sw) << 4), hi[0], hi[1], hi[2], hi[3]);
            sts128(base + (((uint32_t)(4 + half * 2 + k) ^ sw) << 4), lo[0], lo[1], lo[2], lo[3]);
        }
        if (half == 0) B.unit[row] = scale_value(e) * 0.0078125f * a.scale_log2;
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = B.tmem;
    // this CTA's pages: [p0, p0 + cnt)
    const int n_all = (B.hi + PAGE - 1) / PAGE;
    const int p0 = (int)((long long)n_all * split / splits), cnt = (int)((long long)n_all * (split + 1) / splits) - p0;

    if (warp < 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_CTRL));
        if (warp == 0) {
            // -------------------------------------------------------- pages
            const int32_t *table = a.table + b * a.table_stride + p0;
            int id = 0, su = 0, j = 0;
            for (; j < cnt; ++j) {
                if ((j & 31) == 0) {  // ids and scales of the next 32 pages, one a lane
                    id = 0;
                    su = 0xFFFF;
                    if (j + lane < cnt) {
                        id = table[j + lane];
                        if (id < 0 || id >= a.n_pages) {  // no such page: its tokens count as NaN
                            atomicOr(a.status, RESS_STATUS_CACHE_RANGE);
                            id = 0;
                        } else {
                            su = a.K.scale[id * a.K.scale_stride + h] | (a.V.scale[id * a.V.scale_stride + h] << 8);
                        }
                    }
                }
                const int idj = __shfl_sync(0xffffffffu, id, j & 31), suj = __shfl_sync(0xffffffffu, su, j & 31);
                const int ks = j % NK, cs = j % NC;
                if (j >= NK && !wait_bar_warp(&B.k_empty[ks], (j / NK - 1) & 1, abort_flag, a.status)) break;
                if (j >= NC && !wait_bar_warp(&B.c_empty[cs], (j / NC - 1) & 1, abort_flag, a.status)) break;
                if (lane == 0) {
                    B.info[j % INFO] = suj;
                    mbar_expect_tx(&B.k_full[ks], BLOCK_BYTES);
                    tma_load_4d(sK + ks * BLOCK_BYTES, &tm_k, &B.k_full[ks], 0, 0, h, idj);
                    mbar_expect_tx(&B.c_full[cs], BLOCK_BYTES);
                    bulk_load(sC + cs * BLOCK_BYTES, a.V.codes + idj * a.V.page_stride + h * a.V.head_stride, BLOCK_BYTES,
                              &B.c_full[cs]);
                }
                __syncwarp();
            }
            // the last copy into each stage lands before the CTA may exit
            static_assert(NK == NC, "one drain for both rings");
            for (int s = 0; s < NK && s < j; ++s) {
                const int last = j - 1 - ((j - 1 - s) % NK);
                const uint64_t t0 = globaltimer();
                while (!(mbar_try_wait(smem_u32(&B.k_full[s]), (last / NK) & 1) &&
                         mbar_try_wait(smem_u32(&B.c_full[s]), (last / NC) & 1)) &&
                       globaltimer() - t0 < TIMEOUT_NS) {
                }
            }
        } else if (warp == 1) {
            // -------------------------------------------------------- S
            // The whole warp runs the loop, so that descriptors stay in uniform
            // registers; one elected lane issues.
            if (cnt > 0) {
                bool ok = true;
                const bool elected = elect_one();
                const uint64_t dq = make_desc(sQ, 16, 1024, LAYOUT_SW128), dk = make_desc(sK, 16, 512, LAYOUT_SW64);
                int ks = 0, kphase = 0, pb = 0;
                for (int j = 0; ok && j < cnt; ++j) {
                    const int sb = j & 1;
                    if (!wait_bar_warp(&B.k_full[ks], kphase, abort_flag, a.status)) break;
                    for (int t = 0; t < nt; ++t) {
                        if (j >= 2 && !wait_bar_warp(&B.s_free[t][sb], ((j - 2) >> 1) & 1, abort_flag, a.status)) {
                            ok = false;
                            break;
                        }
                        // P_j takes the place of P_{j-NP}, whose product must be done
                        if (j >= NP && !wait_bar_warp(&B.o_full[t][pb], ((j - NP) / NP) & 1, abort_flag, a.status)) {
                            ok = false;
                            break;
                        }
                        fence_after();
                        if (elected) {
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk)  // hi, hi, lo, lo against K's two halves
                                mma_e4m3(tmem + t * 128 + sb * 64, dq + t * (Q_BYTES >> 4) + kk * 2,
                                         dk + ks * (BLOCK_BYTES >> 4) + (kk & 1) * 2, kk > 0 ? 1u : 0u);
                            mma_commit(&B.s_full[t][sb]);
                        }
                        __syncwarp();
                    }
                    if (ok && elected) mma_commit(&B.k_empty[ks]);
                    if (++ks == NK) {
                        ks = 0;
                        kphase ^= 1;
                    }
                    if (++pb == NP) pb = 0;
                }
                if (elected) {
                    mma_commit(&B.s_done);  // every MMA of this thread completes before tensor memory is freed
                    const uint64_t t0 = globaltimer();
                    while (!mbar_try_wait(smem_u32(&B.s_done), 0) && globaltimer() - t0 < TIMEOUT_NS) {
                    }
                }
            }
        } else if (warp == 2) {
            // -------------------------------------------------------- O
            if (cnt > 0) {
                bool ok = true;
                const bool elected = elect_one();
                // B = [V | ones]: the second 128-byte atom along N lies LBO bytes past the
                // first; a step of 2048 bytes in V moves the start and the distance
                const uint64_t dp = make_desc(smem_u32(smem + OFF_P), 16, 1024, LAYOUT_SW128);
                const uint64_t dv = make_desc(sV, sOnes - sV, 1024, LAYOUT_SW128);
                constexpr uint64_t V_STEP = (2048 >> 4) - ((uint64_t)(2048 >> 4) << 16);
                int vs = 0, vphase = 0, pb = 0, pphase = 0;
                for (int j = 0; ok && j < cnt; ++j) {
                    if (!wait_bar_warp(&B.v_full[vs], vphase, abort_flag, a.status)) break;
                    for (int t = 0; t < nt; ++t) {
                        if (!wait_bar_warp(&B.p_full[t][pb], pphase, abort_flag, a.status)) {
                            ok = false;
                            break;
                        }
                        fence_after();
                        if (elected) {
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk)
                                mma_f16(tmem + 256 + t * 128, dp + (t * NP + pb) * (P_BYTES >> 4) + kk * 2,
                                        dv + (uint64_t)(vs * 4 + kk) * V_STEP, IDESC_O, (j | kk) ? 1u : 0u);
                            mma_commit(&B.o_full[t][pb]);
                        }
                        __syncwarp();
                    }
                    if (ok && elected) mma_commit(&B.v_empty[vs]);
                    if (++vs == NV) {
                        vs = 0;
                        vphase ^= 1;
                    }
                    if (++pb == NP) {
                        pb = 0;
                        pphase ^= 1;
                    }
                }
                if (elected) {
                    mma_commit(&B.pv_done);
                    const uint64_t t0 = globaltimer();
                    while (!mbar_try_wait(smem_u32(&B.pv_done), 0) && globaltimer() - t0 < TIMEOUT_NS) {
                    }
                }
            }
        } else if (warp >= 4) {
            // -------------------------------------------------------- V to bf16
            const int c = tid - 128;
            for (int j = 0; j < cnt; ++j) {
                const int cs = j % NC, vs = j % NV;
                if (!wait_bar(&B.c_full[cs], (j / NC) & 1, abort_flag, a.status)) break;
                const int uv = (B.info[j % INFO] >> 8) & 255, uk = B.info[j % INFO] & 255;
                uint4 w[2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(w[i].x), "=r"(w[i].y), "=r"(w[i].z), "=r"(w[i].w)
                                 : "r"(sC + cs * BLOCK_BYTES + (c + 128 * i) * 16));
                if (j >= NV && !wait_bar(&B.v_empty[vs], (j / NV - 1) & 1, abort_flag, a.status)) break;
                // 2^(uv - 127 + 120), in two steps where that is beyond bf16; a page of NaN
                // scale becomes zeros here and NaN in P, where it meets only rows that see it
                const bool nan = uv == 255 || uk == 255;
                const uint32_t f = nan ? 0u : pow2_bf16x2(min(uv - 7, 120));
                const bool big = !nan && uv > 127;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int key = (c + 128 * i) >> 2, qd = c & 3;
                    uint32_t o[8];
                    codes_to_bf16(w[i].x, f, o[0], o[1]);
                    codes_to_bf16(w[i].y, f, o[2], o[3]);
                    codes_to_bf16(w[i].z, f, o[4], o[5]);
                    codes_to_bf16(w[i].w, f, o[6], o[7]);
                    if (big) {
                        const uint32_t g = pow2_bf16x2(uv - 127);
#pragma unroll
                        for (int k = 0; k < 8; ++k) o[k] = mul_bf16x2(o[k], g);
                    }
                    const uint32_t row = sV + vs * V_BYTES + key * 128, sw = (uint32_t)(key & 7);
                    sts128(row + (((uint32_t)(2 * qd) ^ sw) << 4), o[0], o[1], o[2], o[3]);
                    sts128(row + (((uint32_t)(2 * qd + 1) ^ sw) << 4), o[4], o[5], o[6], o[7]);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(&B.v_full[vs]);
                mbar_arrive(&B.c_empty[cs]);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFT));
        // ------------------------------------------------------------ softmax
        const int tile = (warp - 8) >> 3, w = warp & 7;
        if (tile < nt) {
            const int lane0 = (w & 3) * 32 + (w >> 2) * 16;  // first tensor-memory lane of this warp
            const int r = lane0 + (lane & 15), col0 = (lane >> 4) * 32;
            Row rc;
            rc.tS = tmem + tile * 128;
            rc.tO = tmem + 256 + tile * 128;
            rc.lane_addr = (uint32_t)lane0 << 16;
            rc.sP = smem_u32(smem + OFF_P) + tile * NP * P_BYTES;
            rc.prow = (uint32_t)r * 128u;
            rc.rsw = (uint32_t)(r & 7);
            rc.ch0 = (uint32_t)(col0 >> 3);
            rc.col0 = col0;
            rc.o_full = B.o_full[tile];
            rc.s_free = B.s_free[tile];
            rc.abort_flag = abort_flag;
            rc.status = a.status;
            const float unit = B.unit[tile * TILE + r];
            const int lim = B.lim[tile * TILE + r], lo = B.lo[tile];
            uint32_t poff[4];  // swizzled places of this thread's four pieces in its row of P
#pragma unroll
            for (int ch = 0; ch < 4; ++ch) poff[ch] = rc.sP + rc.prow + (((rc.ch0 + (uint32_t)ch) ^ rc.rsw) << 4);
            float m = -INFINITY;
            bool ok = true, ready = false;
            int pb = 0;
            for (int j = 0; j < cnt; ++j) {
                const int sb = j & 1;
                if (!__all_sync(0xffffffffu, ready) &&
                    !wait_bar_warp(&B.s_full[tile][sb], (j >> 1) & 1, abort_flag, a.status)) {
                    ok = false;
                    break;
                }
                fence_after();
                const int su = B.info[j % INFO], base = (p0 + j) * PAGE;
                const float c =
                    unit * ((su & 255) == 255 || su >= 0xFF00 ? __int_as_float(0x7FC00000) : scale_value(su & 255));
                if (j > 0 && base + PAGE <= lo) {
                    uint32_t sv[32];
                    tmem_ld_half32(rc.tS + sb * 64 + rc.lane_addr, sv);
                    tmem_wait_ld();
                    fence_before();
                    mbar_arrive(&B.s_free[tile][sb]);
                    float a0 = -INFINITY, a1 = -INFINITY, a2 = -INFINITY, a3 = -INFINITY;
#pragma unroll
                    for (int t = 0; t < 32; t += 8) {
                        a0 = fmaxf(a0, fmaxf(__uint_as_float(sv[t]), __uint_as_float(sv[t + 1])));
                        a1 = fmaxf(a1, fmaxf(__uint_as_float(sv[t + 2]), __uint_as_float(sv[t + 3])));
                        a2 = fmaxf(a2, fmaxf(__uint_as_float(sv[t + 4]), __uint_as_float(sv[t + 5])));
                        a3 = fmaxf(a3, fmaxf(__uint_as_float(sv[t + 6]), __uint_as_float(sv[t + 7])));
                    }
                    float mx = fmaxf(fmaxf(a0, a1), fmaxf(a2, a3));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16)) * c;  // with the row's other half
                    const bool grow = mx > m + RESCALE_THRESH;
                    if (__any_sync(0xffffffffu, grow)) {
                        const float m_new = grow ? mx : m;
                        const int pj = j - 1;
                        if (!wait_bar_warp(&B.o_full[tile][pj % NP], (pj / NP) & 1, abort_flag, a.status)) {
                            ok = false;
                            break;
                        }
                        fence_after();
                        rescale_o(rc.tO, rc.lane_addr, grow ? ex2(m - m_new) : 1.0f);
                        m = m_new;
                    }
                    const float bias = -m;
                    // S_{j+1} is looked for now and used after this page's exponentials
                    ready = mbar_test_wait(smem_u32(&B.s_full[tile][sb ^ 1]), ((j + 1) >> 1) & 1);
#pragma unroll
                    for (int ch = 0; ch < 4; ++ch) {
                        uint32_t hh[4];
#pragma unroll
                        for (int t = 0; t < 8; t += 2) {
                            float x0, x1;
                            fma2(x0, x1, __uint_as_float(sv[ch * 8 + t]), __uint_as_float(sv[ch * 8 + t + 1]), c, bias);
                            hh[t >> 1] = pack_bf16(ex2(x0), ex2(x1));
                        }
                        sts128(poff[ch] + pb * P_BYTES, hh[0], hh[1], hh[2], hh[3]);
                    }
                    fence_before();
                } else {
                    ready = false;
                    m = step_general(rc, j, lim - base, c, m);
                    if (m != m) {
                        ok = false;
                        break;
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(&B.p_full[tile][pb]);
                pb = pb == NP - 1 ? 0 : pb + 1;
            }
            if (ok && cnt > 0) {
                ok = wait_bar_warp(&B.o_full[tile][(cnt - 1) % NP], ((cnt - 1) / NP) & 1, abort_flag, a.status);
                fence_after();
            }
            float l = 0.0f, o[32];
            if (ok && cnt > 0) {
                uint32_t ov[32];
                const uint32_t lv = tmem_ld_rowsum(rc.tO + HD + rc.lane_addr);
                tmem_ld_half32(rc.tO + rc.lane_addr, ov);
                tmem_wait_ld();
                l = __uint_as_float(lv);
#pragma unroll
                for (int i = 0; i < 32; i += 4) {  // columns of V came in pairs (0, 2), (1, 3)
                    o[i] = __uint_as_float(ov[i]);
                    o[i + 1] = __uint_as_float(ov[i + 2]);
                    o[i + 2] = __uint_as_float(ov[i + 1]);
                    o[i + 3] = __uint_as_float(ov[i + 3]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = 0.0f;
            }
            const int row = r0 + tile * TILE + r;
            const bool in = row < a.rows;
            const long long at = in ? row_at(a, b, h, row, a.o_sb, a.o_st, a.o_sh) + col0 : 0;
            if (splits == 1) {
                if (in) store_row(a, at, o, l == 0.0f ? 0.0f : 1.0f / l);
            } else {
                const long long group = ((long long)b * gridDim.y + h) * row_ctas * TILES + cta * TILES + tile;
                float *slot = a.partial + (group * splits * TILE + r) * PART_ROW;  // this row of piece 0
                float *mine = slot + (long long)split * TILE * PART_ROW;
#pragma unroll
                for (int i = 0; i < 32; i += 4)
                    *reinterpret_cast<float4 *>(mine + col0 + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                if (col0 == 0) {
                    mine[HD] = m;
                    mine[HD + 1] = l;
                }
                __threadfence();
                asm volatile("bar.sync %0, 256;" ::"r"(1 + tile) : "memory");
                if (r == 0 && col0 == 0) B.join[tile] = atomicAdd(&a.arrived[group], 1) == splits - 1;
                asm volatile("bar.sync %0, 256;" ::"r"(1 + tile) : "memory");
                if (B.join[tile] && in) {
                    __threadfence();
                    float mm = -INFINITY;
                    for (int s = 0; s < splits; ++s) mm = fmaxf(mm, __ldcg(slot + (long long)s * TILE * PART_ROW + HD));
                    const float mb = mm == -INFINITY ? 0.0f : mm;
                    float sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0.0f;
                    for (int s = 0; s < splits; ++s) {
                        const float *p = slot + (long long)s * TILE * PART_ROW;
                        const float f = ex2(__ldcg(p + HD) - mb);
                        sum = fmaf(__ldcg(p + HD + 1), f, sum);
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 v = __ldcg(reinterpret_cast<const float4 *>(p + col0 + i));
                            o[i] = fmaf(v.x, f, o[i]);
                            o[i + 1] = fmaf(v.y, f, o[i + 1]);
                            o[i + 2] = fmaf(v.z, f, o[i + 2]);
                            o[i + 3] = fmaf(v.w, f, o[i + 3]);
                        }
                    }
                    store_row(a, at, o, sum == 0.0f ? 0.0f : 1.0f / sum);
                }
            }
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 3)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// CTAs that the pages of one (256 rows, head, stream) are split over: the
// fewest waves of CTAs per piece, pieces of four pages or more.
static int pick_splits(long long ctas, long long table_width) {
    int best = 1;
    double cost = 1e30;
    for (int s = 1; s <= SPLIT_MAX && (s == 1 || s * 4 <= table_width); ++s) {
        const double waves = (double)((ctas * s + 147) / 148);
        const double c = waves / s * (s > 1 ? 1.03 : 1.0) + 0.002 * s;
        if (c < cost) {
            cost = c;
            best = s;
        }
    }
    return best;
}

}  // namespace many

static long long row_ctas(long long rows) { return (rows + many::TILE * many::TILES - 1) / (many::TILE * many::TILES); }

size_t many_workspace(int B, int Hkv, long long rows, long long table_width) {
    const long long ctas = row_ctas(rows) * Hkv * B;
    const int splits = many::pick_splits(ctas, table_width);
    if (splits == 1) return 0;
    return (size_t)ctas * many::TILES * (splits * many::TILE * many::PART_ROW * sizeof(float) + 16);
}

int launch_many(const AttnArgs &args, int B, int Hkv, void *workspace, cudaStream_t stream) {
    AttnArgs a = args;
    const long long rc = row_ctas(a.rows), ctas = rc * Hkv * B;
    const int splits = many::pick_splits(ctas, a.table_width);
    if (rc * splits > INT_MAX) return RESS_E_SHAPE;
    if (splits > 1) {
        if (!workspace || ((uintptr_t)workspace & 15)) return RESS_E_ARG;
        a.arrived = reinterpret_cast<int32_t *>(workspace);
        a.partial = reinterpret_cast<float *>(reinterpret_cast<char *>(workspace) + ctas * many::TILES * 16);
        if (cudaMemsetAsync(a.arrived, 0, (size_t)ctas * many::TILES * sizeof(int32_t), stream) != cudaSuccess)
            return RESS_E_LAUNCH;
    }
    auto enc = tc::get_encode();
    if (!enc) return RESS_E_NO_DEVICE;
    CUtensorMap tm;
    cuuint64_t dims[4] = {HD, PAGE, (cuuint64_t)Hkv, (cuuint64_t)a.n_pages};
    cuuint64_t strides[3] = {HD, (cuuint64_t)a.K.head_stride, (cuuint64_t)a.K.page_stride};
    cuuint32_t box[4] = {HD, PAGE, 1, 1}, es[4] = {1, 1, 1, 1};
    if (enc(&tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, a.K.codes, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return RESS_E_ARG;
    set_smem_attr((const void *)many::many_kernel, many::SMEM);
    many::many_kernel<<<dim3((unsigned)(rc * splits), (unsigned)Hkv, (unsigned)B), many::NT, many::SMEM, stream>>>(
        tm, a, (int)rc, splits);
    return cudaGetLastError() == cudaSuccess ? RESS_OK : RESS_E_LAUNCH;
}

}  // namespace cache
}  // namespace ress

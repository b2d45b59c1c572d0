// cache_attn_tc.cu -- attention of many queries over the paged 8-bit cache on
// the tensor cores (cache_attn.cuh has the definition).
//
// One CTA per 256 rows of a (stream, key/value head), as two tiles of 128
// that share every page of keys and values; 16 warps:
//   warp 0       loads pages: K blocks (TMA, 64B-swizzled), V blocks (bulk);
//   warp 1       issues S = Q K^T, tcgen05.mma kind::f8f6f4.  K's codes are an
//                operand as they lie in the cache.  q is split into two e4m3
//                parts, q = hi + lo, so S takes four K = 32 steps: hi and lo
//                against the same K, which is what bf16 would take.  4 + 4
//                significant bits are as many as bf16 has, down to 2^-9 of the
//                row's largest element; smaller ones meet e4m3's subnormals and
//                err by up to 2^-17 of it, which over 64 dims is below what P is
//                rounded by.  Scales are applied to S.
//   warp 2       issues O += P V, kind::f16 in bf16, P from tensor memory (an
//                MMA of 128 x 80 x 16 takes 40 cycles so, 52 with P in shared
//                memory).  N = 80: sixteen columns of ones give the row sums.
//   warp 3       allocates tensor memory.
//   warps 4-7    turn V's codes into bf16 (exact: the scale is a power of two)
//                in the 128B-swizzled layout that the MMA reads, once for both
//                tiles.
//   warps 8-15   softmax, four warps a tile, one thread per row: a page's 64
//                scores in registers (two loads of the 32x32b shape, which
//                reads tensor memory twice as fast as the 16-lane shapes), no
//                exchange between threads, P back to tensor memory.  The
//                running maximum moves only when it grows by more than 2^8, so
//                O in tensor memory is rarely rescaled.
// Scores are double-buffered.  The bound is the exponential unit, 16 a cycle
// and SM: 1024 cycles a page for both tiles, against 708 cycles of MMAs; a page
// takes about 1700.  The rest are the waits, loads and stores of one tile,
// which queue behind the other's exponentials, and the supply of instructions:
// what is rare is out of line, and the loop over pages is kept short.
// 5,496 queries x 43,968 tokens x 16 heads, each frame seeing those up to its
// own: 1644 us, 573 TFLOP/s of the products that no mask hides; 1374 x 10,992:
// 143 us, 435 (a CTA's start and join weigh more).
// (Measured on the first at one and the same split: 1684 us so; 1782 with the
// masked path in the loop; 1860 with the scores read again in pieces of 16;
// 1835 with steps of 128 keys; 2070 with the next page's scores loaded ahead;
// 1845 with the two tiles' exponentials taking turns; a polynomial for a part
// of the exponentials gained nothing.)
// P is rounded to bf16 (2^-8) for the MMA, numerator and denominator alike: tf32
// has half the rate and takes twice P's way to tensor memory, and fp16 has not
// the range of V's scales.  Against 64 bits that is 0.55e-3 of an output, whose
// own rounding to bf16 is 1.6e-3; everything else is fp32.
// When the tiles are too few for the GPU the pages are split over several
// CTAs; the one that finishes last joins the pieces in page order, so the
// result does not depend on the order of arrival.  (With a piece's rows each
// contiguous, 272 bytes a thread, the single frame took 158 us.)
// Every wait is bounded (tcgen05.cuh).  No TMA multicast.
#include "cache_attn.cuh"

namespace ress {
namespace cache {
namespace many {

using namespace tc;

constexpr int NT = 512, TILE = 128, TILES = 2;
constexpr int NK = 8, NC = 8, NV = 4;  // rings: K, V codes, V in bf16
constexpr int INFO = 32;               // scales of pages in flight: more than any ring is deep
constexpr int REGS_CTRL = 64, REGS_SOFT = 192;
static_assert(256 * REGS_CTRL + 256 * REGS_SOFT <= NT * 128, "register split above the launch's registers");
constexpr int Q_BYTES = TILE * 128, V_BYTES = PAGE * 128, ONES_BYTES = 16 * 128;
constexpr int OFF_Q = 0;
constexpr int OFF_K = OFF_Q + TILES * Q_BYTES;
constexpr int OFF_C = OFF_K + NK * BLOCK_BYTES;
constexpr int OFF_V = OFF_C + NC * BLOCK_BYTES;
constexpr int OFF_ONES = OFF_V + NV * V_BYTES;
constexpr int SMEM = OFF_ONES + ONES_BYTES + 1024;
static_assert(V_BYTES == 4 * 2048, "four K = 16 slices a page");
static_assert(SMEM + 4096 <= 227 * 1024, "shared memory");
// Tensor memory columns: S (two buffers of 64 a tile), O (64 and the 16 row-sum columns), P (bf16 pairs)
constexpr uint32_t COL_S = 0, COL_O = 256, COL_P = 448, O_STRIDE = 96;
constexpr float RESCALE_THRESH = 8.0f;
constexpr int SPLIT_MAX = 8, PART_ROW = HD + 4;  // a partial row: O, maximum, sum

// D f32; A, B e4m3, K-major; N = 64.  And D f32; A, B bf16, B MN-major; N = 80.
constexpr uint32_t IDESC_S = (1u << 4) | ((64u >> 3) << 17) | ((128u >> 4) << 24);
constexpr uint32_t IDESC_O =
    (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((80u >> 3) << 17) | ((128u >> 4) << 24);

struct Bars {
    uint64_t k_full[NK], k_empty[NK], c_full[NC], c_empty[NC], v_full[NV], v_empty[NV];
    uint64_t s_full[TILES][2], s_free[TILES][2], p_full[TILES], o_full[TILES];
    uint64_t s_done, pv_done;
    uint32_t tmem;
    int abort_flag, hi, lo[TILES], join[TILES];
    int nan_seen;  // a NaN code among the values that some row sees
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
__device__ __forceinline__ float max3(uint32_t a, uint32_t b, uint32_t c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
    return r;
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
// 2^120 and the page's scale is exact.  NaN codes become 480: what they do to
// the rows that see them is put in at the end (nan_dims).
__device__ __forceinline__ void codes_to_bf16(uint32_t w, uint32_t f, uint32_t &even, uint32_t &odd) {
    even = mul_bf16x2(((w << 8) & 0x80008000u) | ((w & 0x007F007Fu) << 4), f);
    odd = mul_bf16x2((w & 0x80008000u) | ((w & 0x7F007F00u) >> 4), f);
}
// 2^e as a bf16 pair
__device__ __forceinline__ uint32_t pow2_bf16x2(int e) { return (uint32_t)((e + 127) << 7) * 0x00010001u; }

// Tensor memory to registers and back: lane = row, n columns.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
        "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
        "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
__device__ __forceinline__ uint32_t tmem_ld1(uint32_t taddr) {
    uint32_t v;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(v) : "r"(taddr));
    return v;
}
// O += P V with P (A) in tensor memory.
__device__ __forceinline__ void mma_pv(uint32_t d, uint32_t p, uint64_t b, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(p), "l"(b), "r"(IDESC_O), "r"(acc));
}

// This thread's row of O, row sum included, times alpha.  Out of line, as
// everything rare is: the loop over pages has to fit the instruction cache
// (unrolled by two with the masked path inline it ran at 2330 cycles a page).
__device__ __noinline__ void rescale_o(uint32_t tO, float alpha) {
#pragma unroll 1
    for (int c = 0; c < HD + 16; c += 8) {
        uint32_t o[8];
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]), "=r"(o[4]), "=r"(o[5]), "=r"(o[6]), "=r"(o[7])
                     : "r"(tO + c));
        tmem_wait_ld();
#pragma unroll
        for (int t = 0; t < 8; ++t) o[t] = __float_as_uint(__uint_as_float(o[t]) * alpha);
        asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(tO + c), "r"(o[0]),
                     "r"(o[1]), "r"(o[2]), "r"(o[3]), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7])
                     : "memory");
    }
    tmem_wait_st();
}

// A wait whose usual case, the phase complete, is one probe.
__device__ __noinline__ bool wait_slow(uint64_t *bar, uint32_t parity, volatile int *abort_flag, int32_t *status) {
    return wait_bar_warp(bar, parity, abort_flag, status);
}
__device__ __forceinline__ bool wait_quick(uint64_t *bar, uint32_t parity, volatile int *abort_flag, int32_t *status) {
    if (__all_sync(0xffffffffu, mbar_try_wait(smem_u32(bar), parity))) return true;
    return wait_slow(bar, parity, abort_flag, status);
}

// What the out-of-line step needs of its thread.
struct Row {
    uint32_t tS, tO, tP;
    uint64_t *s_free, *o_full;
    volatile int *abort_flag;
    int32_t *status;
};

// Page j, of which the row sees the first `seen` keys; c is the factor of its
// scores.  Takes the running maximum and returns the new one, NaN when a wait
// failed.  The scores are there; P and its barrier are the caller's.
__device__ __noinline__ float step_masked(const Row &rc, int j, int seen, float c, float m) {
    uint32_t p[32];
    float mx = -INFINITY;
#pragma unroll 1
    for (int h = 0; h < 64; h += 32) {
        uint32_t sv[32];
        tmem_ld32(rc.tS + (j & 1) * 64 + h, sv);
        tmem_wait_ld();
#pragma unroll
        for (int t = 0; t < 32; ++t)
            if (h + t < seen) mx = fmaxf(mx, __uint_as_float(sv[t]));
    }
    mx = mx == -INFINITY ? mx : mx * c;
    const bool grow = mx > m + RESCALE_THRESH;  // m = -inf: whenever a key is seen
    const float m_new = grow ? mx : m;
    const float bias = m_new == -INFINITY ? 0.0f : -m_new;
#pragma unroll
    for (int h = 0; h < 64; h += 32) {
        uint32_t sv[32];
        tmem_ld32(rc.tS + (j & 1) * 64 + h, sv);
        tmem_wait_ld();
#pragma unroll
        for (int t = 0; t < 32; t += 2) {  // a hidden key is 0 even where the factor is 0 or NaN
            const float x0 = ex2(fmaf(__uint_as_float(sv[t]), c, bias)), x1 = ex2(fmaf(__uint_as_float(sv[t + 1]), c, bias));
            p[(h + t) >> 1] = pack_bf16(h + t < seen ? x0 : 0.0f, h + t + 1 < seen ? x1 : 0.0f);
        }
    }
    fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(rc.s_free + (j & 1));
    if (j > 0) {
        if (!wait_bar_warp(rc.o_full, (j - 1) & 1, rc.abort_flag, rc.status)) return __int_as_float(0x7fffffff);
        fence_after();
        if (__any_sync(0xffffffffu, grow)) rescale_o(rc.tO, grow ? ex2(m - m_new) : 1.0f);
    }
    tmem_st32(rc.tP, p);
    return m_new;
}

// A row to the output, times inv.
__device__ __forceinline__ void store_row(const AttnArgs &a, long long at, const float (&o)[HD], float inv) {
    if (a.out_bf16) {
        uint4 *p = reinterpret_cast<uint4 *>(reinterpret_cast<__nv_bfloat16 *>(a.out) + at);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            p[i] = make_uint4(pack_bf16(o[8 * i] * inv, o[8 * i + 1] * inv), pack_bf16(o[8 * i + 2] * inv, o[8 * i + 3] * inv),
                              pack_bf16(o[8 * i + 4] * inv, o[8 * i + 5] * inv),
                              pack_bf16(o[8 * i + 6] * inv, o[8 * i + 7] * inv));
    } else {
        float4 *p = reinterpret_cast<float4 *>(reinterpret_cast<float *>(a.out) + at);
#pragma unroll
        for (int i = 0; i < 16; ++i)
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
            mbar_init(&B.c_empty[i], 4);
        }
        for (int i = 0; i < NV; ++i) {
            mbar_init(&B.v_full[i], 4);
            mbar_init(&B.v_empty[i], 1);
        }
        for (int t = 0; t < TILES; ++t) {
            for (int i = 0; i < 2; ++i) {
                mbar_init(&B.s_full[t][i], 1);
                mbar_init(&B.s_free[t][i], TILE / 32);
            }
            mbar_init(&B.p_full[t], TILE / 32);
            mbar_init(&B.o_full[t], 1);
            B.lo[t] = INT_MAX;
        }
        mbar_init(&B.s_done, 1);
        mbar_init(&B.pv_done, 1);
        B.abort_flag = 0;
        B.hi = 0;
        B.nan_seen = 0;
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
        const int most = __reduce_max_sync(0xffffffffu, l), least = __reduce_min_sync(0xffffffffu, l >= 0 ? l : INT_MAX);
        if (tid % 32 == 0) {
            atomicMax(&B.hi, most);
            atomicMin(&B.lo[tid / TILE], least);
        }
    } else {
        // q of one row a thread: scaled by a power of two to [128, 256), split into two e4m3 parts
        const int row = tid - TILES * TILE;
        uint4 u[8] = {};
        if (r0 + row < a.rows) {
            const uint4 *p = reinterpret_cast<const uint4 *>(a.q + row_at(a, b, h, r0 + row, a.q_sb, a.q_st, a.q_sh));
#pragma unroll
            for (int k = 0; k < 8; ++k) u[k] = __ldg(p + k);
        }
        uint32_t am = 0;
        const uint32_t *w = reinterpret_cast<const uint32_t *>(u);
#pragma unroll
        for (int k = 0; k < 32; ++k) am = max(am, max((w[k] << 16) & 0x7FFFFFFFu, w[k] & 0x7FFF0000u));
        const int e = max((int)(am >> 23), 8);  // 2^(134 - e) stays in range, for a zero row as well
        const float f = row_inverse(e) * 128.0f;
        const uint32_t base = sQ + (row / TILE) * Q_BYTES + (row % TILE) * 128;
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // 16 dims: one 16-byte piece of each part
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                float x[4];
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
                lo[n] = e4m3x4(x[0] - f01.x, x[1] - f01.y, x[2] - f23.x, x[3] - f23.y);
            }
            const uint32_t sw = (uint32_t)(row & 7);
            sts128(base + (((uint32_t)k ^ sw) << 4), hi[0], hi[1], hi[2], hi[3]);
            sts128(base + (((uint32_t)(4 + k) ^ sw) << 4), lo[0], lo[1], lo[2], lo[3]);
        }
        B.unit[row] = scale_value(e) * 0.0078125f * a.scale_log2;
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
                int ks = 0, kphase = 0;
                for (int j = 0; ok && j < cnt; ++j) {
                    const int sb = j & 1;
                    if (!wait_bar_warp(&B.k_full[ks], kphase, abort_flag, a.status)) break;
                    for (int t = 0; t < nt; ++t) {
                        if (j >= 2 && !wait_bar_warp(&B.s_free[t][sb], ((j - 2) >> 1) & 1, abort_flag, a.status)) {
                            ok = false;
                            break;
                        }
                        fence_after();
                        if (elected) {
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk)  // hi, hi, lo, lo against K's two halves
                                mma_e4m3(tmem + COL_S + t * 128 + sb * 64, dq + t * (Q_BYTES >> 4) + kk * 2,
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
                const uint64_t dv = make_desc(sV, sOnes - sV, 1024, LAYOUT_SW128);
                constexpr uint64_t V_STEP = (2048 >> 4) - ((uint64_t)(2048 >> 4) << 16);
                int vs = 0, vphase = 0;
                for (int j = 0; ok && j < cnt; ++j) {
                    if (!wait_bar_warp(&B.v_full[vs], vphase, abort_flag, a.status)) break;
                    for (int t = 0; t < nt; ++t) {
                        if (!wait_bar_warp(&B.p_full[t], j & 1, abort_flag, a.status)) {
                            ok = false;
                            break;
                        }
                        fence_after();
                        if (elected) {
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk)
                                mma_pv(tmem + COL_O + t * O_STRIDE, tmem + COL_P + t * 32 + kk * 8,
                                       dv + (uint64_t)(vs * 4 + kk) * V_STEP, (j | kk) ? 1u : 0u);
                            mma_commit(&B.o_full[t]);
                        }
                        __syncwarp();
                    }
                    if (ok && elected) mma_commit(&B.v_empty[vs]);
                    if (++vs == NV) {
                        vs = 0;
                        vphase ^= 1;
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
                if (!wait_bar_warp(&B.c_full[cs], (j / NC) & 1, abort_flag, a.status)) break;
                const int uv = (B.info[j % INFO] >> 8) & 255, uk = B.info[j % INFO] & 255;
                uint4 w[2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(w[i].x), "=r"(w[i].y), "=r"(w[i].z), "=r"(w[i].w)
                                 : "r"(sC + cs * BLOCK_BYTES + (c + 128 * i) * 16));
                if (j >= NV && !wait_bar_warp(&B.v_empty[vs], (j / NV - 1) & 1, abort_flag, a.status)) break;
                // 2^(uv - 127 + 120), in two steps where that is beyond bf16; a page of NaN
                // scale becomes zeros here and NaN in P, where it meets only rows that see it
                const bool nan = uv == 255 || uk == 255;
                const uint32_t f = nan ? 0u : pow2_bf16x2(min(uv - 7, 120));
                const bool big = !nan && uv > 127;
                uint32_t nans = 0;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int key = (c + 128 * i) >> 2, qd = c & 3;
                    if ((p0 + j) * PAGE + key < B.hi)
                        nans |= nan_codes(w[i].x) | nan_codes(w[i].y) | nan_codes(w[i].z) | nan_codes(w[i].w);
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
                if (nans) B.nan_seen = 1;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&B.v_full[vs]);
                    mbar_arrive(&B.c_empty[cs]);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFT));
        // ------------------------------------------------------------ softmax
        const int tile = (warp - 8) >> 2, quad = warp & 3;
        if (tile < nt) {
            const int r = quad * 32 + lane;
            const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
            const uint32_t tS = lanes + COL_S + tile * 128, tO = lanes + COL_O + tile * O_STRIDE;
            const uint32_t tP = lanes + COL_P + tile * 32;
            const float unit = B.unit[tile * TILE + r];
            const int lim = B.lim[tile * TILE + r], lo = B.lo[tile];
            const Row rc{tS, tO, tP, B.s_free[tile], &B.o_full[tile], abort_flag, a.status};
            // K's scales of 32 pages, one a lane (NaN where V's is, or the page number is
            // bad), times the row's unit: the factor of a page's scores is at hand before
            // they are
            const int32_t *table = a.table + b * a.table_stride + p0;
            auto fetch = [&](int first) {
                int u = 255;
                if (first + lane < cnt) {
                    const int id = table[first + lane];
                    if (id >= 0 && id < a.n_pages) {
                        u = a.K.scale[id * a.K.scale_stride + h];
                        if (a.V.scale[id * a.V.scale_stride + h] == 255) u = 255;
                    }
                }
                return scale_value(u);
            };
            float scales = fetch(0), scales_next = fetch(32);
            float m = -INFINITY;
            bool ok = true;
            const int hot = max(0, min(cnt, lo / PAGE - p0));  // pages that every row sees whole
            int j = 0;
#pragma unroll 1
            for (; j < hot; ++j) {
                if ((j & 31) == 0 && j > 0) {
                    scales = scales_next;
                    scales_next = fetch(j + 32);
                }
                const float c = unit * __shfl_sync(0xffffffffu, scales, j & 31);
                if (!wait_quick(&B.s_full[tile][j & 1], (j >> 1) & 1, abort_flag, a.status)) {
                    ok = false;
                    break;
                }
                fence_after();
                uint32_t sv[64], p[32];
                tmem_ld32(tS + (j & 1) * 64, sv);
                tmem_ld32(tS + (j & 1) * 64 + 32, sv + 32);
                tmem_wait_ld();
                fence_before();
                if (lane == 0) mbar_arrive(&B.s_free[tile][j & 1]);  // of the whole warp, which waited
                float top[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) top[t] = max3(sv[3 * t], sv[3 * t + 1], sv[3 * t + 2]);
#pragma unroll
                for (int t = 12; t < 60; t += 8)
#pragma unroll
                    for (int k = 0; k < 4; ++k) top[k] = max3(__float_as_uint(top[k]), sv[t + 2 * k], sv[t + 2 * k + 1]);
                top[0] = max3(__float_as_uint(top[0]), sv[60], sv[61]);
                top[1] = max3(__float_as_uint(top[1]), sv[62], sv[63]);
                const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * c;
                const bool grow = mx > m + RESCALE_THRESH;  // m = -inf: at once
                const float m_new = grow ? mx : m;
#pragma unroll
                for (int t = 0; t < 64; t += 2) {
                    float x0, x1;
                    fma2(x0, x1, __uint_as_float(sv[t]), __uint_as_float(sv[t + 1]), c, -m_new);
                    p[t >> 1] = pack_bf16(ex2(x0), ex2(x1));
                }
                // P_{j-1} has been read, and O may be rescaled, once its product is done
                if (j > 0) {
                    if (!wait_quick(&B.o_full[tile], (j - 1) & 1, abort_flag, a.status)) {
                        ok = false;
                        break;
                    }
                    fence_after();
                    if (__any_sync(0xffffffffu, grow)) rescale_o(tO, grow ? ex2(m - m_new) : 1.0f);
                }
                m = m_new;
                tmem_st32(tP, p);
                tmem_wait_st();
                fence_before();
                if (lane == 0) mbar_arrive(&B.p_full[tile]);
            }
#pragma unroll 1
            for (; ok && j < cnt; ++j) {  // a limit cuts these for some row
                if ((j & 31) == 0 && j > 0) {
                    scales = scales_next;
                    scales_next = fetch(j + 32);
                }
                const float c = unit * __shfl_sync(0xffffffffu, scales, j & 31);
                ok = wait_quick(&B.s_full[tile][j & 1], (j >> 1) & 1, abort_flag, a.status);
                if (!ok) break;
                fence_after();
                m = step_masked(rc, j, lim - (p0 + j) * PAGE, c, m);
                ok = m == m;
                if (!ok) break;
                tmem_wait_st();
                fence_before();
                if (lane == 0) mbar_arrive(&B.p_full[tile]);
            }
            if (ok && cnt > 0) {
                ok = wait_bar_warp(&B.o_full[tile], (cnt - 1) & 1, abort_flag, a.status);
                fence_after();
            }
            float l = 0.0f, o[HD];
            if (ok && cnt > 0) {
                uint32_t ov[HD];
                const uint32_t lv = tmem_ld1(tO + HD);
                tmem_ld32(tO, ov);
                tmem_ld32(tO + 32, ov + 32);
                tmem_wait_ld();
                l = __uint_as_float(lv);
#pragma unroll
                for (int i = 0; i < HD; i += 4) {  // columns of V came in pairs (0, 2), (1, 3)
                    o[i] = __uint_as_float(ov[i]);
                    o[i + 1] = __uint_as_float(ov[i + 2]);
                    o[i + 2] = __uint_as_float(ov[i + 1]);
                    o[i + 3] = __uint_as_float(ov[i + 3]);
                }
                if (*(volatile int *)&B.nan_seen) {
                    const uint64_t nan = nan_dims(a.V.codes + h * a.V.head_stride, a.V.page_stride, table - p0, a.n_pages, p0, 1, cnt, lim);
#pragma unroll
                    for (int i = 0; i < HD; ++i)
                        if (nan >> i & 1) o[i] = NAN;
                }
            } else {
#pragma unroll
                for (int i = 0; i < HD; ++i) o[i] = 0.0f;
            }
            const int row = r0 + tile * TILE + r;
            const bool in = row < a.rows;
            const long long at = in ? row_at(a, b, h, row, a.o_sb, a.o_st, a.o_sh) : 0;
            if (splits == 1) {
                if (in) store_row(a, at, o, l == 0.0f ? 0.0f : 1.0f / l);
            } else {
                const long long group = ((long long)b * gridDim.y + h) * row_ctas * TILES + cta * TILES + tile;
                // a piece: 17 times 128 rows' four floats (O, then maximum and sum), so that
                // a warp's accesses are contiguous
                constexpr int PIECE = TILE * PART_ROW / 4;
                float4 *slot = reinterpret_cast<float4 *>(a.partial) + group * splits * PIECE + r;  // of piece 0
                float4 *mine = slot + split * PIECE;
#pragma unroll
                for (int i = 0; i < HD; i += 4) mine[i / 4 * TILE] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                mine[HD / 4 * TILE] = make_float4(m, l, 0.0f, 0.0f);
                __threadfence();
                asm volatile("bar.sync %0, 128;" ::"r"(1 + tile) : "memory");
                if (r == 0) B.join[tile] = atomicAdd(&a.arrived[group], 1) == splits - 1;
                asm volatile("bar.sync %0, 128;" ::"r"(1 + tile) : "memory");
                if (B.join[tile] && in) {
                    __threadfence();
                    float mm = -INFINITY;
                    for (int s = 0; s < splits; ++s) mm = fmaxf(mm, __ldcg(slot + s * PIECE + HD / 4 * TILE).x);
                    const float mb = mm == -INFINITY ? 0.0f : mm;
                    float sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < HD; ++i) o[i] = 0.0f;
                    for (int s = 0; s < splits; ++s) {
                        const float4 *p = slot + s * PIECE, ml = __ldcg(p + HD / 4 * TILE);
                        const float f = ex2(ml.x - mb);
                        sum = fmaf(ml.y, f, sum);
#pragma unroll
                        for (int i = 0; i < HD; i += 4) {
                            const float4 v = __ldcg(p + i / 4 * TILE);
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

// CTAs that the pages of one (256 rows, head, stream) are split over: the one
// of 1 .. 8 that makes the waves of CTAs shortest, counting a CTA as its pages
// and the fourteen that its start, its partial result and the join cost
// (measured: 13 us, against 0.93 us a page).
static int pick_splits(long long ctas, long long table_width) {
    int best = 1;
    double least = 1e300;
    for (int s = 1; s <= SPLIT_MAX && (s == 1 || s * 4 <= table_width); ++s) {
        const long long waves = (ctas * s + 147) / 148;
        const double cost = waves * ((double)table_width / s + 14.0);
        if (cost < least) {
            least = cost;
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

// cache_attn.cu -- attention of a few queries over the paged 8-bit cache, and
// the C entry for any number (cache_attn.cuh has the definition).
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
// flight.  The codes become fp16 fragments in registers (one conversion per
// two values; e4m3 is exact in fp16):
//   S: B operand = K.  A lane's 16-byte piece of a key row serves the four
//      k-steps; that orders the head dims differently from memory, and the
//      q fragments are loaded in the same order.
//   O: B operand = V, A = P straight from S's accumulators.  Keys are
//      assigned to accumulator columns as n ^ ((n >> 1) & 1) within eight,
//      so that both K's and V's shared-memory reads touch even and odd rows
//      (64-byte rows: two of equal parity meet in a bank).
// The running maximum, sums and O are fp32.  Row scales of q (a power of two
// that brings its largest element to [1, 2)) keep q exact in fp16; P is
// rounded to fp16 after scaling by 2^14 and the page's V scale over the
// largest one seen, so that small probabilities keep their bits.
// The pages are split over the CTAs of a cluster (and the warps of a CTA).
// Each CTA sends its rows' partial results to the shared memory of the row's
// owner, which joins them in CTA order: one launch, no workspace.
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
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
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
    const float inv = scale_inverse(e);
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = half2_bits(x[2 * j] * inv, x[2 * j + 1] * inv);
    return scale_value(e) * a.scale_log2;
}

// HALF: eight rows at most, the tile's upper half is not computed.
template <bool HALF>
__global__ void __launch_bounds__(FEW_NT, 2) few_kernel(const AttnArgs a, int kv_heads) {
    extern __shared__ __align__(128) unsigned char dyn[];
    __shared__ uint64_t full[FEW_WARPS][FEW_RING];
    __shared__ int abort_s;
    __shared__ float part_m[FEW_WARPS][FEW_ROWS], part_l[FEW_WARPS][FEW_ROWS];
    // what the cluster's CTAs send to this one: for its n-th row, one slot per CTA
    __shared__ __align__(16) float inbox[FEW_ROWS * SLOT + FEW_SPLITS * SLOT];
    const int split = blockIdx.x, splits = gridDim.x;
    const int h = blockIdx.y % kv_heads, tile = blockIdx.y / kv_heads, b = blockIdx.z;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int r0 = tile * FEW_ROWS, rows = min(FEW_ROWS, a.rows - r0);
    volatile int *abort_flag = &abort_s;
    if (threadIdx.x < FEW_WARPS * FEW_RING) mbar_init(&full[0][0] + threadIdx.x, 1);
    if (threadIdx.x == 0) abort_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncthreads();
    if (splits > 1) cluster_arrive();  // waited for before the first store into a peer

    // what the rows see
    const int len = stream_len(a, b);
    if (threadIdx.x == 0 && split == 0 && bad_len(a, b)) atomicOr(a.status, RESS_STATUS_CACHE_RANGE);
    int lim[2], lo = INT_MAX, hi = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        lim[i] = row_limit(a, b, len, r0 + g + 8 * i);
        if (lim[i] >= 0) {
            lo = min(lo, lim[i]);
            hi = max(hi, lim[i]);
        }
    }
    if (a.limits != nullptr) {
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
    } else {
        lo = hi = len;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (lim[i] < 0) lim[i] = hi;  // rows past the last: computed, never written

    // this warp's pages: first, first + FEW_WARPS, ... (count of them)
    const int n = (hi + PAGE - 1) / PAGE;
    const int p0 = (int)((long long)n * split / splits), p1 = (int)((long long)n * (split + 1) / splits);
    const int first = p0 + warp, count = p1 > first ? (p1 - first + FEW_WARPS - 1) / FEW_WARPS : 0;
    // page ids and scales, 32 pages at a time: lane i holds page base + i
    const int32_t *table = a.table + b * a.table_stride;
    auto fetch = [&](int base, int &id, int &su) {
        id = 0;
        su = 0;
        const int i = base + lane;
        if (i < count) {
            id = table[first + i * FEW_WARPS];
            if (id < 0 || id >= a.n_pages) {  // no such page: its tokens count as NaN
                atomicOr(a.status, RESS_STATUS_CACHE_RANGE);
                id = 0;
                su = 0xFFFF;
            } else {
                su = a.K.scale[id * a.K.scale_stride + h] | (a.V.scale[id * a.V.scale_stride + h] << 8);
            }
        }
    };
    int id_a, su_a, id_b = 0, su_b = 0;  // batches of even and odd number
    fetch(0, id_a, su_a);
    unsigned char *ring = dyn + warp * FEW_RING * BLOCK_BYTES;
    const uint32_t ring_a = smem_u32(ring);
    const int blocks = 2 * count;
    int fill_slot = 0;  // ring slot of the next block to ask for
    auto issue = [&](int n) {  // block n: K (even) or V of page n / 2; all lanes call it
        const int i = n >> 1, id = __shfl_sync(0xffffffffu, (i & 32) ? id_b : id_a, i & 31);
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
    fetch(32, id_b, su_b);

    uint32_t q0[8], q1[8] = {};
    const float rf0 = load_q16(a, b, h, r0 + g, t, q0);
    float rf1 = 0.0f;
    if (!HALF) rf1 = load_q16(a, b, h, r0 + g + 8, t, q1);

    float o[8][4] = {};
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
    int uref = 0;  // O counts in units of 2^(uref - 127 - P_SHIFT)
    const int kf = 2 * t + (t & 1), kh = 2 * t + 1 - (t & 1);  // keys of a lane's even and odd columns
    const uint32_t koff = (uint32_t)(g ^ ((g >> 1) & 1)) * HD + t * 16;
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
        if ((i & 31) == 0 && i > 0) {
            if (i & 32) fetch(i + 32, id_a, su_a);
            else fetch(i + 32, id_b, su_b);
        }
        const int su = __shfl_sync(0xffffffffu, (i & 32) ? su_b : su_a, i & 31);
        const int uk = su & 255, uv = su >> 8;
        const unsigned char *sk = take();
        if (sk == nullptr) break;
        uint4 kx[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) kx[j] = *reinterpret_cast<const uint4 *>(sk + j * 8 * HD + koff);
        float c[8][4] = {};
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t w = st == 0 ? kx[j].x : st == 1 ? kx[j].y : st == 2 ? kx[j].z : kx[j].w;
                mma_16816(c[j], q0[2 * st], HALF ? 0u : q1[2 * st], q0[2 * st + 1], HALF ? 0u : q1[2 * st + 1],
                          e4m3_to_half2((uint16_t)w), e4m3_to_half2((uint16_t)(w >> 16)));
            }
        done();
        const float fk = scale_value(uk);
        const float c0 = rf0 * fk, c1 = rf1 * fk;
        const int base = (first + i * FEW_WARPS) * PAGE;
        const bool whole = base + PAGE <= lo;
        float x0 = -INFINITY, x1 = -INFINITY;
        if (!whole) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {  // hidden tokens: -inf, whatever lies there
                const int ke = base + 8 * j + kf, ko = base + 8 * j + kh;
                if (ke >= lim[0]) c[j][0] = -INFINITY;
                if (ko >= lim[0]) c[j][1] = -INFINITY;
                if (!HALF && ke >= lim[1]) c[j][2] = -INFINITY;
                if (!HALF && ko >= lim[1]) c[j][3] = -INFINITY;
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x0 = fmaxf(x0, fmaxf(c[j][0], c[j][1]));
            if (!HALF) x1 = fmaxf(x1, fmaxf(c[j][2], c[j][3]));
        }
        // the page's largest score; the factors are not negative (a NaN one shows in the exponentials)
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
        const float n0 = fmaxf(m0, x0 == -INFINITY ? x0 : x0 * c0), b0 = n0 == -INFINITY ? 0.0f : n0;
        float al0 = ex2(m0 - b0), al1 = 1.0f, b1 = 0.0f;
        m0 = n0;
        if (!HALF) {
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
            const float n1 = fmaxf(m1, x1 == -INFINITY ? x1 : x1 * c1);
            b1 = n1 == -INFINITY ? 0.0f : n1;
            al1 = ex2(m1 - b1);
            m1 = n1;
        }
        l0 *= al0;
        l1 *= al1;
        // a page of larger V scale moves O's unit
        float fv = scale_value(uv);  // NaN stays NaN
        if (uv != 255) {
            if (uv > uref) {
                const float d = scale_value(max(127 + uref - uv, 0));
                al0 *= d;
                al1 *= d;
                uref = uv;
            }
            fv = scale_value(max(127 + P_SHIFT + uv - uref, 0));
        }
        if (__any_sync(0xffffffffu, al0 != 1.0f || al1 != 1.0f)) {
#pragma unroll
            for (int d = 0; d < 8; ++d) {
                o[d][0] *= al0;
                o[d][1] *= al0;
                o[d][2] *= al1;
                o[d][3] *= al1;
            }
        }
        // P: probabilities for the sums, and times the V scale as fp16 fragments
        uint32_t pa[4][4];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float p[4] = {};
            p[0] = ex2(fmaf(c[j][0], c0, -b0));
            p[1] = ex2(fmaf(c[j][1], c0, -b0));
            if (!HALF) {
                p[2] = ex2(fmaf(c[j][2], c1, -b1));
                p[3] = ex2(fmaf(c[j][3], c1, -b1));
            }
            if (!whole) {  // a hidden token is 0 even where a factor is 0 or NaN
                const int ke = base + 8 * j + kf, ko = base + 8 * j + kh;
                if (ke >= lim[0]) p[0] = 0.0f;
                if (ko >= lim[0]) p[1] = 0.0f;
                if (ke >= lim[1]) p[2] = 0.0f;
                if (ko >= lim[1]) p[3] = 0.0f;
            }
            l0 += p[0] + p[1];
            l1 += p[2] + p[3];
#pragma unroll
            for (int e = 0; e < 4; ++e) p[e] *= fv;
            if (!whole && uv == 255) {
                const int ke = base + 8 * j + kf, ko = base + 8 * j + kh;
                if (ke >= lim[0]) p[0] = 0.0f;
                if (ko >= lim[0]) p[1] = 0.0f;
                if (ke >= lim[1]) p[2] = 0.0f;
                if (ko >= lim[1]) p[3] = 0.0f;
            }
            pa[j >> 1][2 * (j & 1)] = half2_bits(p[0], p[1]);
            pa[j >> 1][2 * (j & 1) + 1] = HALF ? 0u : half2_bits(p[2], p[3]);
        }
        const unsigned char *sv = take();
        if (sv == nullptr) break;
#pragma unroll
        for (int st = 0; st < 4; ++st) {
            const unsigned char *va = sv + st * 16 * HD + g * 8;
            uint2 v0 = *reinterpret_cast<const uint2 *>(va + kf * HD), v1 = *reinterpret_cast<const uint2 *>(va + kh * HD);
            uint2 v2 = *reinterpret_cast<const uint2 *>(va + (8 + kf) * HD);
            uint2 v3 = *reinterpret_cast<const uint2 *>(va + (8 + kh) * HD);
            if (base + PAGE > len) {  // slots past the stream's end hold anything, NaN codes too
                const int e = len - base - 16 * st;
                if (kf >= e) v0 = make_uint2(0, 0);
                if (kh >= e) v1 = make_uint2(0, 0);
                if (8 + kf >= e) v2 = make_uint2(0, 0);
                if (8 + kh >= e) v3 = make_uint2(0, 0);
            }
#pragma unroll
            for (int d = 0; d < 8; d += 2) {
                const uint32_t sel = (d & 2) ? 0x7362u : 0x5140u;
                const uint32_t y0 = d < 4 ? __byte_perm(v0.x, v1.x, sel) : __byte_perm(v0.y, v1.y, sel);
                const uint32_t y1 = d < 4 ? __byte_perm(v2.x, v3.x, sel) : __byte_perm(v2.y, v3.y, sel);
                mma_16816(o[d], pa[st][0], pa[st][1], pa[st][2], pa[st][3], e4m3_to_half2((uint16_t)y0),
                          e4m3_to_half2((uint16_t)y1));
                mma_16816(o[d + 1], pa[st][0], pa[st][1], pa[st][2], pa[st][3], e4m3_to_half2((uint16_t)(y0 >> 16)),
                          e4m3_to_half2((uint16_t)(y1 >> 16)));
            }
        }
        done();
    }
    // copies in flight land before their ring is used again (all have, unless a wait ran out)
    for (int s = 0; s < min(issued, FEW_RING); ++s) {
        const int last = issued - 1 - ((issued - 1 - s) % FEW_RING);
        const uint64_t t0 = globaltimer();
        while (!mbar_try_wait(smem_u32(&full[warp][s]), (last / FEW_RING) & 1) && globaltimer() - t0 < TIMEOUT_NS) {
        }
    }
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    if (t == 0) {
        part_m[warp][g] = m0;
        part_l[warp][g] = l0;
        part_m[warp][g + 8] = m1;
        part_l[warp][g + 8] = l1;
    }
    __syncthreads();
    // the warps' O meet in the ring, 4 KB a warp
    float *po = reinterpret_cast<float *>(dyn) + warp * FEW_ROWS * HD;
    const float unit = scale_value(uref), down = scale_value(127 - P_SHIFT);
#pragma unroll
    for (int half = 0; half < (HALF ? 1 : 2); ++half)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int d = 0; d < 8; d += 4)
                *reinterpret_cast<float4 *>(po + (g + 8 * half) * HD + 16 * t + 8 * e + d) =
                    make_float4(o[d][2 * half + e] * down * unit, o[d + 1][2 * half + e] * down * unit,
                                o[d + 2][2 * half + e] * down * unit, o[d + 3][2 * half + e] * down * unit);
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
    const long long groups = (long long)tiles * Hkv * B;
    // CTAs for about two per SM, as long as there is a page for each warp
    int splits = 1;
    while (splits < FEW_SPLITS && groups * splits * 2 <= 148 * 2 && splits * 2 * FEW_WARPS <= a.table_width) splits *= 2;
    auto kern = a.rows <= 8 ? few_kernel<true> : few_kernel<false>;
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

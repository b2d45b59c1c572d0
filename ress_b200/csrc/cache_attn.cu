// cache_attn.cu -- attention of a few queries over the paged 8-bit cache, and
// the C entry for any number (cache_attn.cuh has the definition).
#include "cache_attn.cuh"

namespace ress {
namespace cache {

using namespace tc;

// ------------------------------------------------------------------ few rows
// Up to 16 rows a tile, on mma.sync.m16n8k16: with so few rows the bound is
// the bytes of the cache, and the 128-row tensor-core tiles would be empty.
// Each warp takes pages of its own: K and V blocks (4 KB each) arrive by
// bulk copies in a ring of the warp's, so the warps never wait for one
// another before the end.  The codes become fp16 fragments in registers (one
// conversion per two values; e4m3 is exact in fp16):
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
// The pages are split over the CTAs of a cluster (and the warps of a CTA);
// the partial results meet in distributed shared memory, so one launch does
// it all without a workspace.
constexpr int FEW_ROWS = 16, FEW_WARPS = 4, FEW_STAGES = 3;
constexpr int FEW_NT = FEW_WARPS * 32;
constexpr int FEW_SMEM = FEW_WARPS * FEW_STAGES * 2 * BLOCK_BYTES;
constexpr int P_SHIFT = 14;
// Rows of a (stream, key/value head) up to which this kernel runs.
constexpr int FEW_MAX_ROWS = 32;

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}
// shared memory of another CTA of the cluster
__device__ __forceinline__ uint32_t peer_addr(uint32_t a, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}
__device__ __forceinline__ float peer_f32(uint32_t a) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ float4 peer_f32x4(uint32_t a) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

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
__global__ void __launch_bounds__(FEW_NT) few_kernel(const AttnArgs a, int kv_heads) {
    extern __shared__ __align__(128) unsigned char dyn[];
    __shared__ uint64_t full[FEW_WARPS][FEW_STAGES];
    __shared__ int abort_s;
    __shared__ float part_m[FEW_WARPS][FEW_ROWS], part_l[FEW_WARPS][FEW_ROWS];
    const int split = blockIdx.x, splits = gridDim.x;
    const int h = blockIdx.y % kv_heads, tile = blockIdx.y / kv_heads, b = blockIdx.z;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int r0 = tile * FEW_ROWS;
    volatile int *abort_flag = &abort_s;
    if (threadIdx.x == 0) {
        abort_s = 0;
        for (int w = 0; w < FEW_WARPS; ++w)
            for (int s = 0; s < FEW_STAGES; ++s) mbar_init(&full[w][s], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (split == 0 && bad_len(a, b)) atomicOr(a.status, RESS_STATUS_CACHE_RANGE);
    }
    __syncthreads();

    // what the rows see
    const int len = stream_len(a, b);
    int lim[2], lo = INT_MAX, hi = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        lim[i] = row_limit(a, b, len, r0 + g + 8 * i);
        if (lim[i] >= 0) {
            lo = min(lo, lim[i]);
            hi = max(hi, lim[i]);
        }
    }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (lim[i] < 0) lim[i] = hi;  // rows past the last: computed, never written

    uint32_t q0[8], q1[8] = {};
    const float rf0 = load_q16(a, b, h, r0 + g, t, q0);
    float rf1 = 0.0f;
    if (!HALF) rf1 = load_q16(a, b, h, r0 + g + 8, t, q1);

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
    fetch(32, id_b, su_b);
    const uint32_t ring = smem_u32(dyn) + warp * FEW_STAGES * 2 * BLOCK_BYTES;
    auto issue = [&](int i) {  // all lanes call it
        const int id = __shfl_sync(0xffffffffu, (i & 32) ? id_b : id_a, i & 31);
        if (lane == 0) {
            const int s = i % FEW_STAGES;
            const uint32_t dst = ring + s * 2 * BLOCK_BYTES;
            mbar_expect_tx(&full[warp][s], 2 * BLOCK_BYTES);
            bulk_load(dst, a.K.codes + id * a.K.page_stride + h * a.K.head_stride, BLOCK_BYTES, &full[warp][s]);
            bulk_load(dst + BLOCK_BYTES, a.V.codes + id * a.V.page_stride + h * a.V.head_stride, BLOCK_BYTES,
                      &full[warp][s]);
        }
    };
    const int ahead = min(count, FEW_STAGES);
    for (int i = 0; i < ahead; ++i) issue(i);

    float o[8][4] = {};
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
    int uref = 0;  // O counts in units of 2^(uref - 127 - P_SHIFT)
    const int kf = 2 * t + (t & 1), kh = 2 * t + 1 - (t & 1);  // keys of a lane's even and odd columns
    const uint32_t koff = (uint32_t)(g ^ ((g >> 1) & 1)) * HD + t * 16;
    int issued = ahead;
    for (int i = 0; i < count; ++i) {
        const int s = i % FEW_STAGES;
        // the batch two ahead replaces the one just used up
        if ((i & 31) == 0 && i > 0) {
            if (i & 32) fetch(i + 32, id_a, su_a);
            else fetch(i + 32, id_b, su_b);
        }
        const int su = __shfl_sync(0xffffffffu, (i & 32) ? su_b : su_a, i & 31);
        const int uk = su & 255, uv = su >> 8;
        if (!wait_bar_warp(&full[warp][s], (i / FEW_STAGES) & 1, abort_flag, a.status)) break;
        const uint32_t sk = ring + s * 2 * BLOCK_BYTES, sv = sk + BLOCK_BYTES;
        float c[8][4];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            c[j][0] = c[j][1] = c[j][2] = c[j][3] = 0.0f;
            const uint4 kx = lds128(sk + j * 8 * HD + koff);
            const uint32_t kw[4] = {kx.x, kx.y, kx.z, kx.w};
#pragma unroll
            for (int st = 0; st < 4; ++st)
                mma_16816(c[j], q0[2 * st], HALF ? 0u : q1[2 * st], q0[2 * st + 1], HALF ? 0u : q1[2 * st + 1],
                          e4m3_to_half2((uint16_t)kw[st]), e4m3_to_half2((uint16_t)(kw[st] >> 16)));
        }
        const float fk = scale_value(uk);
        const float c0 = rf0 * fk, c1 = rf1 * fk;
        const int base = (first + i * FEW_WARPS) * PAGE;
        const bool whole = base + PAGE <= lo;
        float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int ke = base + 8 * j + kf, ko = base + 8 * j + kh;
            c[j][0] = whole || ke < lim[0] ? c[j][0] * c0 : -INFINITY;
            c[j][1] = whole || ko < lim[0] ? c[j][1] * c0 : -INFINITY;
            x0 = fmaxf(x0, fmaxf(c[j][0], c[j][1]));
            if (!HALF) {
                c[j][2] = whole || ke < lim[1] ? c[j][2] * c1 : -INFINITY;
                c[j][3] = whole || ko < lim[1] ? c[j][3] * c1 : -INFINITY;
                x1 = fmaxf(x1, fmaxf(c[j][2], c[j][3]));
            }
        }
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
        const float n0 = fmaxf(m0, x0), b0 = n0 == -INFINITY ? 0.0f : n0;
        float al0 = ex2(m0 - b0), al1 = 1.0f, b1 = 0.0f;
        m0 = n0;
        if (!HALF) {
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
            const float n1 = fmaxf(m1, x1);
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
#pragma unroll
        for (int st = 0; st < 4; ++st) {
            uint32_t pa[4] = {};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float *cc = c[2 * st + e];
                const int ke = base + 8 * (2 * st + e) + kf, ko = base + 8 * (2 * st + e) + kh;
                const float pe = ex2(cc[0] - b0), po = ex2(cc[1] - b0);
                l0 += pe + po;
                // a hidden token is 0 even in a page of NaN scale
                pa[2 * e] = half2_bits(whole || ke < lim[0] ? pe * fv : 0.0f, whole || ko < lim[0] ? po * fv : 0.0f);
                if (!HALF) {
                    const float qe = ex2(cc[2] - b1), qo = ex2(cc[3] - b1);
                    l1 += qe + qo;
                    pa[2 * e + 1] =
                        half2_bits(whole || ke < lim[1] ? qe * fv : 0.0f, whole || ko < lim[1] ? qo * fv : 0.0f);
                }
            }
            const uint32_t va = sv + st * 16 * HD + g * 8;
            uint2 v0 = lds64(va + kf * HD), v1 = lds64(va + kh * HD);
            uint2 v2 = lds64(va + (8 + kf) * HD), v3 = lds64(va + (8 + kh) * HD);
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
                mma_16816(o[d], pa[0], pa[1], pa[2], pa[3], e4m3_to_half2((uint16_t)y0), e4m3_to_half2((uint16_t)y1));
                mma_16816(o[d + 1], pa[0], pa[1], pa[2], pa[3], e4m3_to_half2((uint16_t)(y0 >> 16)),
                          e4m3_to_half2((uint16_t)(y1 >> 16)));
            }
        }
        __syncwarp();
        if (issued < count) issue(issued++);
    }
    // copies in flight land before their ring is used again (all have, unless a wait ran out)
    for (int s = 0; s < min(issued, FEW_STAGES); ++s) {
        const int last = issued - 1 - ((issued - 1 - s) % FEW_STAGES);
        const uint64_t t0 = globaltimer();
        while (!mbar_try_wait(smem_u32(&full[warp][s]), (last / FEW_STAGES) & 1) && globaltimer() - t0 < TIMEOUT_NS) {
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
    // the warps' O meet in the ring (4 KB a warp), then the CTA's in its first 4 KB
    float *po = reinterpret_cast<float *>(dyn) + warp * FEW_ROWS * HD;
    const float unit = scale_value(uref), down = scale_value(127 - P_SHIFT);
#pragma unroll
    for (int d = 0; d < 8; ++d) {
        po[g * HD + 16 * t + d] = o[d][0] * down * unit;
        po[g * HD + 16 * t + 8 + d] = o[d][1] * down * unit;
        po[(g + 8) * HD + 16 * t + d] = o[d][2] * down * unit;
        po[(g + 8) * HD + 16 * t + 8 + d] = o[d][3] * down * unit;
    }
    __syncthreads();
    __shared__ float cta_m[FEW_ROWS], cta_l[FEW_ROWS];
    const int rows = min(FEW_ROWS, a.rows - r0);
    float *co = reinterpret_cast<float *>(dyn);
    for (int it = threadIdx.x; it < rows * 16; it += FEW_NT) {
        const int r = it >> 4, d = (it & 15) * 4;
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
        *reinterpret_cast<float4 *>(co + r * HD + d) = acc;  // warp 0's place, read by this thread alone
        if (d == 0) {
            cta_m[r] = mm;
            cta_l[r] = l;
        }
    }
    if (splits > 1) cluster_sync();
    else __syncthreads();
    for (int it = split * FEW_NT + threadIdx.x; it < rows * 16; it += splits * FEW_NT) {
        const int r = it >> 4, d = (it & 15) * 4;
        float4 acc;
        float l;
        if (splits > 1) {
            const uint32_t am = smem_u32(&cta_m[r]), al = smem_u32(&cta_l[r]), ao = smem_u32(co + r * HD + d);
            float mm = -INFINITY;
            for (int s = 0; s < splits; ++s) mm = fmaxf(mm, peer_f32(peer_addr(am, s)));
            const float mb = mm == -INFINITY ? 0.0f : mm;
            acc = make_float4(0.f, 0.f, 0.f, 0.f);
            l = 0.0f;
            for (int s = 0; s < splits; ++s) {
                const float f = ex2(peer_f32(peer_addr(am, s)) - mb);
                const float4 v = peer_f32x4(peer_addr(ao, s));
                acc.x += f * v.x;
                acc.y += f * v.y;
                acc.z += f * v.z;
                acc.w += f * v.w;
                l += f * peer_f32(peer_addr(al, s));
            }
        } else {
            acc = *reinterpret_cast<const float4 *>(co + r * HD + d);
            l = cta_l[r];
        }
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
    }
    if (splits > 1) cluster_sync();  // peers read this CTA's shared memory until here
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
    // CTAs for about two per SM, as long as each has a few pages a warp
    int splits = 1;
    while (splits < 16 && groups * splits * 2 <= 148 * 2 && splits * 2 * FEW_WARPS * 2 <= a.table_width) splits *= 2;
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
    if (g.q_heads <= 0 || g.q_heads % H != 0) return RESS_E_ARG;
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

// int8.cu -- a Linear layer in 8-bit integers: y = (x8 w8^T) sx[m] sw[n] + b.
//
// Weights are int8 with one fp32 scale per output channel, laid out once.
// Activations are quantised per token within the call:
//     sx = max|x| * RN(1/127),   x8 = rint(x / sx)      (x8 = 0 for a zero row)
// Products and sums are exact in int32 (K <= 2^17), so the result depends on
// neither tiles nor order; the scales, the bias and the optional GELU
// (y/2 (1 + erf(y/sqrt 2))) are applied in fp32 and the result is rounded
// once to the output's type.
#include "common.cuh"
#include "prologue.cuh"
#include "tcgen05.cuh"

namespace ress {
namespace i8 {

constexpr float RCP127 = (float)(1.0 / 127.0);

struct LinArgs {
    const int8_t *w;      // (N, K)
    const float *w_scale; // (N)
    const float *bias;    // (N) or null
    void *out;            // (M, N), rows out_st apart
    long long out_st;
    int M, N, K;
    int gelu;
};

// The scale of a row from the bits of its largest magnitude; a row that is
// not finite gets a NaN scale, so that its outputs are NaN.
__device__ __forceinline__ float row_scale(uint32_t amax_bits) {
    return amax_bits >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : __fmul_rn(__uint_as_float(amax_bits), RCP127);
}
__device__ __forceinline__ int round_s8(float x) {
    int r;
    asm("cvt.rni.sat.s8.f32 %0, %1;" : "=r"(r) : "f"(x));
    return r;
}
// How a row's values become codes: x / d rounded to the nearest integer, d
// the scale or 1 where that is 0 or NaN.  The quotient is the correctly
// rounded one (div_by in common.cuh, two lanes at a time), the integer the
// low byte of quotient + 1.5 * 2^23.  Scales so small that the division's
// remainder would be subnormal take the plain division and a saturating
// conversion (a subnormal scale can be off by more than a half code).
struct RowQuant {
    float d;
    f32x2 r, nd;
    bool tiny;
};
__device__ __forceinline__ RowQuant row_quant(float scale) {
    const float d = scale > 0.0f ? scale : 1.0f, r = __frcp_rn(d);
    return {d, f2_pack(r, r), f2_pack(-d, -d), d < 7.9e-31f};
}
__device__ __forceinline__ uint2 quant8(const float (&x)[8], const RowQuant &q) {
    uint32_t c[8];
    if (q.tiny) {
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j] = (uint32_t)round_s8(__fdiv_rn(x[j], q.d));
    } else {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const f32x2 a = f2_pack(x[j], x[j + 1]), y = f2_mul_rn(a, q.r);
            const f32x2 z = f2_fma_rn(f2_fma_rn(y, q.nd, a), q.r, y);
            float u, v;
            f2_unpack(f2_add_rn(z, 0x4B4000004B400000ull), u, v);
            c[j] = __float_as_uint(u);
            c[j + 1] = __float_as_uint(v);
        }
    }
    return make_uint2(pack_low_bytes(c[0], c[1], c[2], c[3]), pack_low_bytes(c[4], c[5], c[6], c[7]));
}
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t amax8(const float (&x)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(x[j]) & 0x7FFFFFFFu);
    return m;
}

// GELU of two values: y Phi(y) = max(y, 0) - |y| Phi(-|y|).  log2 Phi(v) is a
// smooth function, here its polynomial of degree 7 on [-6.5, 0] (fitted so that
// Phi's largest error is least: 1.1e-7; below, Phi < 5e-11): one exponential and
// no reciprocal, and packed arithmetic, where the instructions issued bound the
// epilogue (43,968 x 1024 -> 4096 with the quantiser: 196 us; 215 without the
// packing, and 11 more with a rational form of erfc).
__device__ __forceinline__ f32x2 twice(float x) { return f2_pack(x, x); }
__device__ __forceinline__ f32x2 gelu(f32x2 yy) {
    float y0, y1, p0, p1;
    f2_unpack(yy, y0, y1);
    const f32x2 v = f2_pack(fmaxf(-fabsf(y0), -6.5f), fmaxf(-fabsf(y1), -6.5f));
    f32x2 p = twice(-8.481062650e-06f);
    p = f2_fma_rn(p, v, twice(-5.400051305e-05f));
    p = f2_fma_rn(p, v, twice(4.209168255e-04f));
    p = f2_fma_rn(p, v, twice(7.388782687e-03f));
    p = f2_fma_rn(p, v, twice(5.269075559e-02f));
    p = f2_fma_rn(p, v, twice(-4.591532648e-01f));
    p = f2_fma_rn(p, v, twice(1.151110888f));
    p = f2_fma_rn(p, v, twice(-0.9999998808f));
    f2_unpack(p, p0, p1);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(p0));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(p1));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(y0) : "f"(0.0f));  // a NaN stays one
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(y1) : "f"(0.0f));
    return f2_fma_rn(v, f2_pack(p0, p1), f2_pack(y0, y1));
}
// an accumulator times its row's and channel's scales, plus the channel's bias
__device__ __forceinline__ f32x2 scaled(int acc0, int acc1, f32x2 s_row, f32x2 s_w, f32x2 bias) {
    return f2_fma_rn(f2_mul_rn(f2_pack((float)acc0, (float)acc1), s_row), s_w, bias);
}

// Rows to int8 with one scale each: one warp per row, eight values a lane at
// a time.  CH > 0: the row (at most 256 * CH values) stays in registers
// between its maximum and its codes; CH = 0: it is read again.  Bound by HBM
// where the rows are many: 43,968 x 4096 in bf16, 540 MB, 84 us, as fast as a
// copy.  (Quantising inside the product's kernel is slower than both kernels,
// 208 us: by four more warps that feed its operand 371, since every tile of
// channels quantises its rows again; by four more warps that take each row once
// and count it for the tiles that wait 308, since four warps an SM keep too few
// loads in flight.)
constexpr int QUANT_NT = 256;
template <typename T> struct Piece;  // eight values as loaded
template <> struct Piece<__nv_bfloat16> {
    uint4 u;
    __device__ __forceinline__ void load(const __nv_bfloat16 *p) { u = __ldg(reinterpret_cast<const uint4 *>(p)); }
    __device__ __forceinline__ void clear() { u = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[2 * j] = __uint_as_float(w[j] << 16);
            x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
        }
    }
    // bits of the largest magnitude
    __device__ __forceinline__ uint32_t amax() const {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) m = max(m, max((w[j] << 16) & 0x7FFFFFFFu, w[j] & 0x7FFF0000u));
        return m;
    }
};
template <> struct Piece<float> {
    float v[8];
    __device__ __forceinline__ void load(const float *p) { load8(p, v); }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = v[j];
    }
    __device__ __forceinline__ uint32_t amax() const { return amax8(v); }
};

template <typename T, int CH>
__global__ void __launch_bounds__(QUANT_NT) quant_rows_kernel(const T *__restrict__ x, long long x_st, int M, int K,
                                                              int8_t *__restrict__ q, float *__restrict__ scale) {
    // the product's CTAs may start (and set themselves up) once every CTA of this
    // kernel has; they wait for its end before they read anything of it
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const long long m = ((long long)blockIdx.x * QUANT_NT + threadIdx.x) >> 5;
    if (m >= M) return;
    const T *row = x + m * x_st;
    uint32_t am = 0;
    Piece<T> piece[CH > 0 ? CH : 1];
    if constexpr (CH > 0) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int k = i * 256 + lane * 8;
            if (k < K) piece[i].load(row + k);
            else piece[i].clear();
        }
#pragma unroll
        for (int i = 0; i < CH; ++i) am = max(am, piece[i].amax());
    } else {
        for (int k = lane * 8; k < K; k += 256) {
            piece[0].load(row + k);
            am = max(am, piece[0].amax());
        }
    }
    am = __reduce_max_sync(0xffffffffu, am);
    const float s = row_scale(am);
    const RowQuant rq = row_quant(s);
    if (lane == 0) scale[m] = s;
    int8_t *qr = q + m * K;
    float v[8];
    if constexpr (CH > 0) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int k = i * 256 + lane * 8;
            piece[i].get(v);
            if (k < K) *reinterpret_cast<uint2 *>(qr + k) = quant8(v, rq);
        }
    } else {
        for (int k = lane * 8; k < K; k += 256) {
            piece[0].load(row + k);
            piece[0].get(v);
            *reinterpret_cast<uint2 *>(qr + k) = quant8(v, rq);
        }
    }
}

// ------------------------------------------------------------------ few rows
// Up to sixteen tokens: the weights' bytes (and the latency of a launch) are
// the bound.  A CTA takes 16 channels, its eight warps an eighth of K each, as
// mma.sync.m16n8k32 on two channel tiles; a lane's 16-byte piece of a weight
// row serves two k-steps.  The first weights are asked for before anything
// else; meanwhile every CTA quantises the tokens into shared memory (they
// are few, and no second launch is needed).  The warps' int32 sums are
// exact, so their order does not matter.  1 x 1024 -> 4096: 3.4 us from launch
// to launch, of which its 4 MB of weights take 0.65; the rest are the launch
// and two memory latencies.
constexpr int FEW_NT = 256, FEW_WARPS = 8, FEW_M = 16, FEW_N = 16, FEW_AHEAD = 4;
template <typename T, typename O>
__global__ void __launch_bounds__(FEW_NT) few_kernel(const T *__restrict__ x, long long x_st, const LinArgs a) {
    extern __shared__ __align__(16) unsigned char xs[];  // FEW_M rows of Kp + 16 bytes
    __shared__ float sx[FEW_M];
    __shared__ uint32_t top[FEW_WARPS];
    __shared__ int sums[FEW_WARPS][FEW_M][FEW_N + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * FEW_N;
    const int Kp = (a.K + 63) & ~63, pitch = Kp + 16;
    // this warp's 64-wide steps of K
    const int steps = Kp / 64, s0 = steps * warp / FEW_WARPS, s1 = steps * (warp + 1) / FEW_WARPS;
    const int8_t *w0 = a.w + (long long)min(n0 + g, a.N - 1) * a.K + t * 16;
    const int8_t *w1 = a.w + (long long)min(n0 + 8 + g, a.N - 1) * a.K + t * 16;
    auto weight = [&](const int8_t *w, int s) {
        return s < s1 && s * 64 + t * 16 < a.K ? __ldg(reinterpret_cast<const uint4 *>(w + s * 64)) : make_uint4(0, 0, 0, 0);
    };
    uint4 b0[FEW_AHEAD], b1[FEW_AHEAD];
#pragma unroll
    for (int i = 0; i < FEW_AHEAD; ++i) {
        b0[i] = weight(w0, s0 + i);
        b1[i] = weight(w1, s0 + i);
    }
    // `per` warps share a token; rows without one hold anything: their products
    // stay in their own rows, which are not written
    const int per = a.M >= 8 ? 1 : a.M >= 4 ? 2 : a.M >= 2 ? 4 : 8, sub = warp % per;
    for (int r0 = 0; r0 < a.M; r0 += FEW_WARPS / per) {
        const int r = r0 + warp / per;
        const T *row = x + (long long)min(r, a.M - 1) * x_st;
        uint32_t am = 0;
        Piece<T> p;
        for (int k = sub * 256 + lane * 8; k < a.K; k += 256 * per) {
            p.load(row + k);
            am = max(am, p.amax());
        }
        am = __reduce_max_sync(0xffffffffu, am);
        if (per > 1) {
            if (lane == 0) top[warp] = am;
            __syncthreads();
            for (int i = 0; i < per; ++i) am = max(am, top[warp - sub + i]);
            __syncthreads();
        }
        const float s = row_scale(am);
        const RowQuant rq = row_quant(s);
        for (int k = sub * 256 + lane * 8; k < Kp; k += 256 * per) {
            uint2 w = make_uint2(0, 0);
            if (k < a.K) {
                float v[8];
                p.load(row + k);
                p.get(v);
                w = quant8(v, rq);
            }
            *reinterpret_cast<uint2 *>(xs + r * pitch + k) = w;
        }
        if (lane == 0 && sub == 0) sx[r] = s;
    }
    __syncthreads();
    int c[2][4] = {};
    for (int s = s0; s < s1; s += FEW_AHEAD) {
#pragma unroll
        for (int i = 0; i < FEW_AHEAD; ++i) {
            if (s + i < s1) {
                const int k = (s + i) * 64 + t * 16;
                const uint4 p = *reinterpret_cast<const uint4 *>(xs + g * pitch + k);
                const uint4 q = *reinterpret_cast<const uint4 *>(xs + (g + 8) * pitch + k);
                mma_s8(c[0], p.x, q.x, p.y, q.y, b0[i].x, b0[i].y);
                mma_s8(c[1], p.x, q.x, p.y, q.y, b1[i].x, b1[i].y);
                mma_s8(c[0], p.z, q.z, p.w, q.w, b0[i].z, b0[i].w);
                mma_s8(c[1], p.z, q.z, p.w, q.w, b1[i].z, b1[i].w);
            }
            b0[i] = weight(w0, s + i + FEW_AHEAD);
            b1[i] = weight(w1, s + i + FEW_AHEAD);
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[warp][g + (i >> 1) * 8][u * 8 + 2 * t + (i & 1)] = c[u][i];
    __syncthreads();
    const int r = threadIdx.x / FEW_N, col = threadIdx.x % FEW_N, n = n0 + col;
    if (r < a.M && n < a.N) {
        int acc = 0;
#pragma unroll
        for (int w = 0; w < FEW_WARPS; ++w) acc += sums[w][r][col];
        f32x2 yy = scaled(acc, acc, twice(sx[r]), twice(a.w_scale[n]), twice(a.bias != nullptr ? a.bias[n] : 0.0f));
        if (a.gelu) yy = gelu(yy);
        float y, same;
        f2_unpack(yy, y, same);
        DT<O>::store(reinterpret_cast<O *>(a.out), (size_t)(r * a.out_st + n), y);
    }
}

template <typename T, typename O>
static int launch_few(const void *x, long long x_st, const LinArgs &a, cudaStream_t s) {
    const size_t smem = (size_t)FEW_M * (((a.K + 63) & ~63) + 16);
    if (smem > 32 * 1024) set_smem_attr((const void *)few_kernel<T, O>, smem);
    few_kernel<T, O><<<(a.N + FEW_N - 1) / FEW_N, FEW_NT, smem, s>>>((const T *)x, x_st, a);
    return cudaGetLastError() == cudaSuccess ? RESS_OK : RESS_E_LAUNCH;
}

// ----------------------------------------------------------------- many rows
// Tiles of 128*CG tokens x BN channels on the tensor cores (tcgen05.mma
// kind::i8, int32 accumulators in tensor memory).  CG = 2 pairs two CTAs of a
// cluster on one tile: each loads its half of the tokens and of the channels,
// so a tile's operands cross from L2 once per pair.  Persistent CTAs (pairs)
// take tiles in turn, channel tiles fastest, so that the CTAs that run
// together share token rows in L2.  Twelve warps:
//   warp 0     loads K slices of 128 bytes (TMA, 128B swizzle) into a ring;
//   warp 1     issues the MMAs (the pair's first CTA only, when paired);
//   warp 2     allocates tensor memory;
//   warps 4-11 epilogue: accumulators of one of two buffers to registers,
//              scales, bias, GELU, one rounding, shared memory, TMA store,
//              while the next tile is accumulated into the other buffer; two
//              warps share a quarter of the rows and take its columns in turn.
// With long K the tensor cores are the bound: 43,968 x 4096 -> 1024 takes 125
// us after the quantiser, 2.95 POP/s.  With K = 1024 a tile's operands from L2
// (256 KB at the 40 to 45 bytes a cycle and SM that all SMs reach together) take
// 6,000 cycles and its MMAs 4,100: 1024 -> 1024 41 us, 2.25 POP/s; with GELU the
// epilogue's 7,000 instructions' cycles are near: 1024 -> 4096 173 us, 2.1 POP/s.
using namespace tc;

template <int CG, int BN, typename O> struct Tile {
    static constexpr int NT = 384, BK = 128;
    static constexpr int A_BYTES = 128 * BK, B_ROWS = BN / CG, B_BYTES = B_ROWS * BK;
    static constexpr int STAGE = A_BYTES + B_BYTES;
    static constexpr int OUT_COLS = 128 / (int)sizeof(O);  // one 128-byte swizzled row
    static constexpr int OUT_BYTES = 32 * 128;             // of a warp: 32 rows
    static constexpr int RING = 180 * 1024;
    static constexpr int NS = RING / STAGE < 8 ? RING / STAGE : 8;
    static constexpr int OFF_OUT = NS * STAGE;
    static constexpr int SMEM = OFF_OUT + 8 * OUT_BYTES + 1024;
    static constexpr uint32_t COLS = 2 * BN;  // two accumulators
    static constexpr uint32_t IDESC =
        (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)((128 * CG) >> 4) << 24);
    static_assert(SMEM <= 227 * 1024 && COLS <= 512 && NS >= 2, "tile does not fit");
};

__device__ __forceinline__ void tma_store_2d(const CUtensorMap *map, uint32_t src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"((uint64_t)map),
                 "r"(src), "r"(x), "r"(y)
                 : "memory");
}
template <int CG> __device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y) {
    if constexpr (CG == 2)
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::
                "r"(dst),
            "l"((uint64_t)map), "r"(bar), "r"(x), "r"(y)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::
                "r"(dst),
            "l"((uint64_t)map), "r"(bar), "r"(x), "r"(y)
            : "memory");
}
template <int CG> __device__ __forceinline__ void mma_int8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    if constexpr (CG == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(acc));
    else
        mma_i8(d, a, b, idesc, acc);
}
// arrives on the barrier at this offset in every CTA of the pair
template <int CG> __device__ __forceinline__ void commit(uint64_t *bar) {
    if constexpr (CG == 2)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                smem_u32(bar)),
            "h"((uint16_t)3)
            : "memory");
    else
        mma_commit(bar);
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t leader_addr(uint32_t a) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(a));
    return r;
}
template <int CG> __device__ __forceinline__ void pair_sync() {
    if constexpr (CG == 2) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
        __syncthreads();
    }
}
// Sixteen rows of 32 columns: a lane gets two columns of two rows of each eight
// columns, so that one load of a channel pair's scales serves several rows.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr));
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr));
}

struct GemmBars {
    uint64_t full[8], empty[8], acc_full[2], acc_free[2];
    float w_scale[2][256], bias[2][256];  // of this tile's and the next one's channels
    uint32_t tmem;
    int abort_flag;
};

template <int CG, int BN, typename O>
__global__ void __launch_bounds__(384, 1) gemm_kernel(const __grid_constant__ CUtensorMap tm_x,
                                                      const __grid_constant__ CUtensorMap tm_w,
                                                      const __grid_constant__ CUtensorMap tm_o, const LinArgs a,
                                                      const float *__restrict__ sx, int tma_out, int32_t *status) {
    using C = Tile<CG, BN, O>;
    extern __shared__ unsigned char raw[];
    __shared__ __align__(16) GemmBars B;
    unsigned char *smem = reinterpret_cast<unsigned char *>(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    const uint32_t ring = smem_u32(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = CG == 2 ? (int)cluster_rank() : 0;
    volatile int *abort_flag = &B.abort_flag;
    const int tiles_n = (a.N + BN - 1) / BN, tiles_m = (a.M + 128 * CG - 1) / (128 * CG);
    const int tiles = tiles_n * tiles_m;
    const int first = blockIdx.x / CG, step = gridDim.x / CG;
    const int nk = (a.K + C::BK - 1) / C::BK;
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::NS; ++i) {
            mbar_init(&B.full[i], 1);
            mbar_init(&B.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&B.acc_full[i], 1);
            mbar_init(&B.acc_free[i], 8 * CG);
        }
        B.abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        if constexpr (CG == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&B.tmem)),
                         "r"(C::COLS)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&B.tmem)),
                         "r"(C::COLS)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    fence_before();
    __syncthreads();
    pair_sync<CG>();  // the peer's barriers exist before anything arrives on them
    fence_after();
    const uint32_t tmem = B.tmem;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the tokens' codes and scales are there

    if (warp == 0) {
        if (lane == 0) {
            int it = 0;
            bool ok = true;
            for (int tile = first; ok && tile < tiles; tile += step) {
                const int m0 = (tile / tiles_n) * 128 * CG + rank * 128, n0 = (tile % tiles_n) * BN + rank * C::B_ROWS;
                for (int k = 0; k < nk; ++k, ++it) {
                    const int s = it % C::NS;
                    if (it >= C::NS && !wait_bar(&B.empty[s], (it / C::NS - 1) & 1, abort_flag, status)) {
                        ok = false;
                        break;
                    }
                    const uint32_t dst = ring + s * C::STAGE;
                    const uint32_t bar = CG == 2 ? leader_addr(smem_u32(&B.full[s])) : smem_u32(&B.full[s]);
                    if (rank == 0) mbar_expect_tx(&B.full[s], CG * C::STAGE);
                    tma_load_2d<CG>(dst, &tm_x, bar, k * C::BK, m0);
                    tma_load_2d<CG>(dst + C::A_BYTES, &tm_w, bar, k * C::BK, n0);
                }
            }
            // the last loads of each stage are seen to have landed (and been
            // consumed, both CTAs') before this CTA may exit
            for (int s = 0; s < C::NS && s < it; ++s) {
                const int last = it - 1 - ((it - 1 - s) % C::NS);
                const uint64_t t0 = globaltimer();
                while (!mbar_try_wait_sleep(smem_u32(&B.empty[s]), (last / C::NS) & 1) &&
                       globaltimer() - t0 < TIMEOUT_NS) {
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            int it = 0, n = 0;
            bool ok = true;
            for (int tile = first; ok && tile < tiles; tile += step, ++n) {
                const int buf = n & 1;
                if (n >= 2 && !wait_bar(&B.acc_free[buf], ((n >> 1) - 1) & 1, abort_flag, status)) break;
                fence_after();
                for (int k = 0; k < nk; ++k, ++it) {
                    const int s = it % C::NS;
                    if (!wait_bar(&B.full[s], (it / C::NS) & 1, abort_flag, status)) {
                        ok = false;
                        break;
                    }
                    fence_after();
                    const uint32_t sa = ring + s * C::STAGE, sb = sa + C::A_BYTES;
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        mma_int8<CG>(tmem + buf * BN, make_desc(sa + kk * 32, 16, 1024, LAYOUT_SW128),
                                     make_desc(sb + kk * 32, 16, 1024, LAYOUT_SW128), C::IDESC, (k | kk) ? 1u : 0u);
                    commit<CG>(&B.empty[s]);
                }
                if (ok) commit<CG>(&B.acc_full[buf]);
            }
        }
    } else if (warp >= 4) {
        const int quad = warp & 3, half = (warp >> 2) - 1;
        unsigned char *out_s = smem + C::OFF_OUT + (warp - 4) * C::OUT_BYTES;
        const uint32_t out_a = smem_u32(out_s);
        int n = 0;
        // one channel's scale and bias a thread and its row's scale, asked for a tile
        // ahead (behind the operands' copies they take microseconds)
        const int ch = threadIdx.x - 128;
        float next_w = 0.0f, next_b = 0.0f, next_s = 0.0f;
        bool aborted = false;
        auto ask = [&](int tile) {
            const int col = (tile % tiles_n) * BN + ch;
            const int m = (tile / tiles_n) * 128 * CG + rank * 128 + quad * 32 + lane;
            const bool in = tile < tiles && ch < BN && col < a.N;
            next_w = in ? __ldg(a.w_scale + col) : 0.0f;
            next_b = in && a.bias != nullptr ? __ldg(a.bias + col) : 0.0f;
            next_s = tile < tiles && m < a.M ? sx[m] : 0.0f;
        };
        ask(first);
        for (int tile = first; tile < tiles; tile += step, ++n) {
            const int buf = n & 1;
            const int m0 = (tile / tiles_n) * 128 * CG + rank * 128 + quad * 32, n0 = (tile % tiles_n) * BN;
            f32x2 s_row[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) s_row[i] = twice(__shfl_sync(~0u, next_s, 8 * i + (lane >> 2)));
            const float *const w_scale = B.w_scale[buf], *const bias = B.bias[buf];
            B.w_scale[buf][ch] = next_w;  // last read two tiles ago, before everyone's last barrier
            B.bias[buf][ch] = next_b;
            ask(tile + step);
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const bool ok = wait_bar_warp(&B.acc_full[buf], (n >> 1) & 1, abort_flag, status);
            if (!ok) aborted = true;  // the barriers above still want every warp
            fence_after();
            const uint32_t tq = tmem + buf * BN + ((uint32_t)(quad * 32) << 16);
#pragma unroll 1
            for (int c = half * C::OUT_COLS; c < BN && !aborted; c += 2 * C::OUT_COLS) {
                if (n0 + c >= a.N) break;
                // the piece written before has been read by its store
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                __syncwarp();
#pragma unroll
                for (int part = 0; part < C::OUT_COLS; part += 32) {
                    uint32_t v[2][16];
                    tmem_ld16(tq + c + part, v[0]);
                    tmem_ld16(tq + c + part + (16u << 16), v[1]);
                    tmem_wait_ld();
                    const int cp = c + part + 2 * (lane & 3), col = n0 + cp;
                    f32x2 y[4][4];  // rows 8 r + lane / 4, columns 8 g + 2 (lane % 4) and the next
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const f32x2 w = *reinterpret_cast<const f32x2 *>(&w_scale[cp + 8 * g]);
                        const f32x2 b = *reinterpret_cast<const f32x2 *>(&bias[cp + 8 * g]);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const uint32_t *const acc = &v[r >> 1][4 * g + 2 * (r & 1)];
                            y[g][r] = scaled((int)acc[0], (int)acc[1], s_row[r], w, b);
                        }
                    }
                    if (a.gelu) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) y[i >> 2][i & 3] = gelu(y[i >> 2][i & 3]);
                    }
                    if (tma_out) {
                        // 16-byte pieces of 32 rows, 128B-swizzled
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            if constexpr (sizeof(O) == 2) {
                                uint32_t x[4];
#pragma unroll
                                for (int r = 0; r < 4; ++r) {
                                    float y0, y1;
                                    f2_unpack(y[g][r], y0, y1);
                                    const __nv_bfloat162 h = __floats2bfloat162_rn(y0, y1);
                                    x[r] = *reinterpret_cast<const uint32_t *>(&h);
                                }
                                const uint32_t at = out_a + lane * 128 + (((part / 8 + g) ^ (lane & 7)) << 4);
                                asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(at),
                                             "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3])
                                             : "memory");
                            } else {
                                const int piece = 2 * g + ((lane & 3) >> 1);
#pragma unroll
                                for (int r = 0; r < 4; ++r) {
                                    const int row = 8 * r + (lane >> 2);
                                    *reinterpret_cast<f32x2 *>(out_s + row * 128 + ((piece ^ (row & 7)) << 4) + (lane & 1) * 8) =
                                        y[g][r];
                                }
                            }
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int row = m0 + 8 * (i & 3) + (lane >> 2), to = col + 8 * (i >> 2);
                            O *const out = reinterpret_cast<O *>(a.out);
                            float y0, y1;
                            f2_unpack(y[i >> 2][i & 3], y0, y1);
                            if (row < a.M && to < a.N) DT<O>::store(out, (size_t)(row * a.out_st + to), y0);
                            if (row < a.M && to + 1 < a.N) DT<O>::store(out, (size_t)(row * a.out_st + to + 1), y1);
                        }
                    }
                }
                if (tma_out) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0 && m0 < a.M) {
                        tma_store_2d(&tm_o, out_a, n0 + c, m0);
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                }
            }
            // the accumulator is read: the issuer may overwrite it
            fence_before();
            __syncwarp();
            if (lane == 0) {
                // Only tensor memory changes hands: this warp's reads of it are complete
                // (tcgen05.wait::ld) and fence::before_thread_sync orders them before the
                // arrival, which the issuer's wait and fence::after_thread_sync take up;
                // ordinary memory needs no order.  A releasing arrive would wait for the
                // loads asked ahead (2,000 to 2,900 cycles of a tile's 10,000).
                if constexpr (CG == 2)
                    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                                     leader_addr(smem_u32(&B.acc_free[buf])))
                                 : "memory");
                else
                    mbar_arrive(&B.acc_free[buf]);
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    pair_sync<CG>();  // neither CTA leaves while the other may still touch its memory
    fence_after();
    if (warp == 2) {
        if constexpr (CG == 2)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLS) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLS) : "memory");
    }
}

// Few tiles: a cluster of S CTAs takes one tile of 128 tokens x 64 channels, each
// a part of K (one SM's copies, at 40 bytes a cycle, bound a tile otherwise).
// Every CTA owns 64 / S of the channels: the others send it their int32 sums of
// those, which are exact, so their order does not matter.
constexpr int SPLIT_NT = 256;
template <int S> struct SplitTile {
    static constexpr int BN = 64, OWN = BN / S, STAGE = (128 + BN) * 128, NS = 6;
    static constexpr int OFF_IN = NS * STAGE;  // sums from every CTA: S x OWN / 4 x 128 rows of four
    static constexpr int SMEM = OFF_IN + 128 * BN * 4 + 1024;
    static constexpr uint32_t IDESC =
        (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((128u >> 4) << 24);
};
template <int S, typename O>
__global__ void __launch_bounds__(SPLIT_NT, 1) split_kernel(const __grid_constant__ CUtensorMap tm_x,
                                                            const __grid_constant__ CUtensorMap tm_w, const LinArgs a,
                                                            const float *__restrict__ sx, int wide_out, int32_t *status) {
    using C = SplitTile<S>;
    extern __shared__ unsigned char raw[];
    __shared__ uint64_t full[C::NS], empty[C::NS], acc_full;
    __shared__ uint32_t tmem_s;
    __shared__ int abort_s;
    unsigned char *smem = reinterpret_cast<unsigned char *>(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    const uint32_t ring = smem_u32(smem), inbox = ring + C::OFF_IN;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int)cluster_rank();
    volatile int *abort_flag = &abort_s;
    const int m0 = blockIdx.z * 128, n0 = blockIdx.y * C::BN;
    const int nk = (a.K + 127) / 128, k0 = nk * rank / S, k1 = nk * (rank + 1) / S;
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::NS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        mbar_init(&acc_full, 1);
        abort_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)), "r"(64)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // started: waited for before the sums are sent
    const uint32_t tmem = tmem_s;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the tokens' codes and scales are there
    if (warp == 0 && lane == 0) {
        for (int k = k0, it = 0; k < k1; ++k, ++it) {
            const int st = it % C::NS;
            if (it >= C::NS && !wait_bar(&empty[st], (it / C::NS - 1) & 1, abort_flag, status)) break;
            mbar_expect_tx(&full[st], C::STAGE);
            tma_load_2d<1>(ring + st * C::STAGE, &tm_x, smem_u32(&full[st]), k * 128, m0);
            tma_load_2d<1>(ring + st * C::STAGE + 128 * 128, &tm_w, smem_u32(&full[st]), k * 128, n0);
        }
    } else if (warp == 1 && lane == 0) {
        bool ok = true;
        for (int k = k0, it = 0; k < k1; ++k, ++it) {
            const int st = it % C::NS;
            ok = wait_bar(&full[st], (it / C::NS) & 1, abort_flag, status);
            if (!ok) break;
            fence_after();
            const uint32_t sa = ring + st * C::STAGE, sb = sa + 128 * 128;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
                mma_int8<1>(tmem, make_desc(sa + kk * 32, 16, 1024, LAYOUT_SW128), make_desc(sb + kk * 32, 16, 1024, LAYOUT_SW128),
                            C::IDESC, (it | kk) ? 1u : 0u);
            commit<1>(&empty[st]);
        }
        if (ok) commit<1>(&acc_full);
    }
    __syncwarp();
    // a warp's 32 rows, and of the 64 channels the first or last 32
    const int row = (warp & 3) * 32 + lane, half = warp >> 2;
    const bool ok = wait_bar_warp(&acc_full, 0, abort_flag, status);
    fence_after();
    uint32_t v[32];
    if (ok) {
        tmem_ld32(tmem + half * 32 + ((uint32_t)((warp & 3) * 32) << 16), v);
        tmem_wait_ld();
    }
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (ok && m0 + row < a.M) {
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
            const int col = half * 32 + i, own = col / C::OWN;
            const uint32_t to = inbox + ((rank * C::OWN + col % C::OWN) / 4 * 128 + row) * 16;
            uint32_t at;
            asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(to), "r"(own));
            asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]),
                         "r"(v[i + 3])
                         : "memory");
        }
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    // meanwhile: the scales of this thread's row and channels
    constexpr int PER = C::OWN / 2;  // channels of a thread, two threads a row
    const int r = threadIdx.x & 127, c0 = (threadIdx.x >> 7) * PER, n = n0 + rank * C::OWN + c0;
    const bool in = m0 + r < a.M;
    const float s_row = in ? sx[m0 + r] : 0.0f;
    float w[PER], b[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        w[i] = n + i < a.N ? __ldg(a.w_scale + n + i) : 0.0f;
        b[i] = n + i < a.N && a.bias != nullptr ? __ldg(a.bias + n + i) : 0.0f;
    }
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (in) {
        int acc[PER] = {};
        const int4 *sums = reinterpret_cast<const int4 *>(smem + C::OFF_IN) + c0 / 4 * 128 + r;
#pragma unroll
        for (int p = 0; p < S; ++p)
#pragma unroll
            for (int i = 0; i < PER; i += 4) {
                const int4 u = sums[(p * C::OWN + i) / 4 * 128];
                acc[i] += u.x;
                acc[i + 1] += u.y;
                acc[i + 2] += u.z;
                acc[i + 3] += u.w;
            }
        O *const out = reinterpret_cast<O *>(a.out) + (size_t)(m0 + r) * a.out_st + n;
        float y[PER];
#pragma unroll
        for (int i = 0; i < PER; i += 2) {
            f32x2 yy = scaled(acc[i], acc[i + 1], twice(s_row), f2_pack(w[i], w[i + 1]), f2_pack(b[i], b[i + 1]));
            if (a.gelu) yy = gelu(yy);
            f2_unpack(yy, y[i], y[i + 1]);
        }
        if (wide_out && n + PER <= a.N) {
#pragma unroll
            for (int i = 0; i < PER; i += 16 / (int)sizeof(O)) {
                if constexpr (sizeof(O) == 2) {
                    uint32_t u[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const __nv_bfloat162 h = __floats2bfloat162_rn(y[i + 2 * k], y[i + 2 * k + 1]);
                        u[k] = *reinterpret_cast<const uint32_t *>(&h);
                    }
                    *reinterpret_cast<uint4 *>(out + i) = make_uint4(u[0], u[1], u[2], u[3]);
                } else {
                    *reinterpret_cast<float4 *>(out + i) = make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (n + i < a.N) DT<O>::store(out, (size_t)i, y[i]);
        }
    }
    // copies in flight have landed (all have been consumed, unless a wait ran out)
    if (warp == 0 && lane == 0 && !ok)
        for (int st = 0; st < min(k1 - k0, C::NS); ++st) {
            const uint64_t t0 = globaltimer();
            while (!mbar_try_wait_sleep(smem_u32(&full[st]), ((k1 - k0 - 1 - st) / C::NS) & 1) && globaltimer() - t0 < TIMEOUT_NS) {
            }
        }
    __syncwarp();
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(64) : "memory");
}

// Rows of `cols` elements, `stride` bytes apart, in boxes of 128 bytes x box_rows.
static bool map_2d(CUtensorMap *m, const void *base, CUtensorMapDataType dt, int elem, long long cols, long long rows,
                   long long stride, int box_rows) {
    auto enc = get_encode();
    if (!enc) return false;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride};
    cuuint32_t box[2] = {(cuuint32_t)(128 / elem), (cuuint32_t)box_rows}, es[2] = {1, 1};
    return enc(m, dt, 2, const_cast<void *>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int CG, int BN, typename O>
static int launch_gemm(const int8_t *x8, const float *sx, const LinArgs &a, int32_t *status, cudaStream_t s) {
    using C = Tile<CG, BN, O>;
    CUtensorMap tx, tw, to;
    if (!map_2d(&tx, x8, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.K, a.M, a.K, 128) ||
        !map_2d(&tw, a.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.K, a.N, a.K, C::B_ROWS))
        return RESS_E_NO_DEVICE;
    const int size = (int)sizeof(O);
    // rows whose stride or start a TMA store cannot take are stored by plain instructions
    const int tma_out = !((uintptr_t)a.out & 15) && !((a.out_st * size) & 15);
    to = tx;
    if (tma_out && !map_2d(&to, a.out, size == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32,
                           size, a.N, a.M, a.out_st * size, 32))
        return RESS_E_NO_DEVICE;
    const long long tiles = (long long)((a.N + BN - 1) / BN) * ((a.M + 128 * CG - 1) / (128 * CG));
    const int slots = 148 / CG;
    auto kern = gemm_kernel<CG, BN, O>;
    set_smem_attr((const void *)kern, C::SMEM);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(CG * (tiles < slots ? tiles : slots)));
    cfg.blockDim = dim3(C::NT);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = CG;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, tx, tw, to, a, sx, tma_out, status) == cudaSuccess ? RESS_OK : RESS_E_LAUNCH;
}

template <int S, typename O>
static int launch_split(const int8_t *x8, const float *sx, const LinArgs &a, int32_t *status, cudaStream_t s) {
    using C = SplitTile<S>;
    CUtensorMap tx, tw;
    if (!map_2d(&tx, x8, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.K, a.M, a.K, 128) ||
        !map_2d(&tw, a.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.K, a.N, a.K, C::BN))
        return RESS_E_NO_DEVICE;
    auto kern = split_kernel<S, O>;
    set_smem_attr((const void *)kern, C::SMEM);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(S, (unsigned)((a.N + C::BN - 1) / C::BN), (unsigned)((a.M + 127) / 128));
    cfg.blockDim = dim3(SPLIT_NT);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = S;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    const int wide_out = !((uintptr_t)a.out & 15) && !((a.out_st * (int)sizeof(O)) & 15);
    return cudaLaunchKernelEx(&cfg, kern, tx, tw, a, sx, wide_out, status) == cudaSuccess ? RESS_OK : RESS_E_LAUNCH;
}

template <typename T>
static int launch_quant(const T *x, long long x_st, int M, int K, int8_t *x8, float *scale, cudaStream_t s) {
    const unsigned blocks = (unsigned)(((long long)M * 32 + QUANT_NT - 1) / QUANT_NT);
    constexpr int MOST = sizeof(T) == 2 ? 16 : 8;  // 64 registers of a row
    auto kern = K <= 1024        ? quant_rows_kernel<T, 4>
                : K <= 2048      ? quant_rows_kernel<T, 8>
                : K <= 256 * MOST ? quant_rows_kernel<T, MOST>
                                  : quant_rows_kernel<T, 0>;
    kern<<<blocks, QUANT_NT, 0, s>>>(x, x_st, M, K, x8, scale);
    return cudaGetLastError() == cudaSuccess ? RESS_OK : RESS_E_LAUNCH;
}

// Tokens up to which every CTA quantises them all sooner than a second kernel
// starts.  Measured, us against the tiles below, 1024 channels: 16 x 1024 4.9
// against 5.5, 16 x 2048 6.4 against 6.7, 16 x 4096 15.5 against 9.2; 8 x 4096 9.5
// against 9.2; 4 x 8192 11.2 against 14.6.
static bool use_few(int M, int K) { return K <= 8192 && (M <= 4 || (M <= FEW_M && M * K <= 32 * 1024)); }
static size_t workspace(int M, int K) {
    return use_few(M, K) ? 0 : ((size_t)M * K + 255) / 256 * 256 + (size_t)M * sizeof(float);
}

// CTAs that share a tile of 128 x 64: as many as leave every CTA an SM (a GPC's
// SMs are not all multiples of four) and a slice of K.  Measured, us with one, two
// and four (quantiser included): 64 x 1024 -> 1024: 7.6, 6.9, 5.9; 165 x 1536 ->
// 1000: 9.7, 8.7, 7.3; 64 x 4096 -> 1024: 16.4, 12.2, 9.5; beyond an SM each: 100 x
// 1024 -> 4096 in four 10.3 (two 7.3, one 7.8), 165 x 1024 -> 3000 in two 11.2
// (one 8.1).
static int pick_split(const LinArgs &a) {
    const long long tiles = (long long)((a.M + 127) / 128) * ((a.N + 63) / 64);
    const int nk = (a.K + 127) / 128;
    return tiles * 4 <= 128 && nk >= 4 ? 4 : tiles * 2 <= 148 && nk >= 2 ? 2 : 1;
}

// The tile (of <pair, 256>, <single, 128>, <single, 64>) whose waves over the
// GPU are estimated to cost least, in cycles.  A K = 128 slice takes the longer
// of its MMAs (an MMA of K = 32 reads 128 + BN rows of 32 bytes at 128 bytes a
// cycle and computes 8192 products a cycle: 128, 64, 48 cycles) and its copies
// (40 bytes a cycle and SM with all SMs copying, as measured; about 80 for a
// few; a tile of 64 channels' smaller slices are no faster than in proportion).
// The epilogue of a wave overlaps the next wave's slices; pairs start and end
// 3000 cycles later.  Measured, us on the three tiles, quantiser included:
// 43,968 x 1024 -> 1024: 64, 83, 132; 1374 x 1024 -> 4096 with GELU: 15.0,
// 15.6, 20.0; 1374 x 4096 -> 1024: 19.5, 18.3, 27.8; 165 x 1536 -> 1000: 10.6,
// 9.3, 8.9 (a pair's tiles of 128 channels: 85, 16.2, 18.8, 9.6).
static int pick_tile(const LinArgs &a) {
    const int cg[3] = {2, 1, 1}, bn[3] = {256, 128, 64}, mma[3] = {128, 64, 48};
    const double slices = (a.K + 127) / 128;
    int best = 0;
    double least = 1e300;
    for (int i = 0; i < 3; ++i) {
        const long long tiles = (long long)((a.M + 128 * cg[i] - 1) / (128 * cg[i])) * ((a.N + bn[i] - 1) / bn[i]);
        const long long slots = 148 / cg[i], waves = (tiles + slots - 1) / slots;
        const double active = (double)((tiles < slots ? tiles : slots) * cg[i]);
        const double rate = active > 74 ? 5920.0 / active : 80.0, bytes = 128.0 * (bn[i] > 64 ? 256 : 192);
        const double slice = bytes / rate > 4 * mma[i] ? bytes / rate : 4 * mma[i];
        const double epilogue = bn[i] * (a.gelu ? 24.0 : 12.0), main = slices * slice;
        const double cost = waves * (main > epilogue ? main : epilogue) + epilogue + (cg[i] > 1 ? 3000.0 : 0.0);
        if (cost < least) {
            least = cost;
            best = i;
        }
    }
    return best;
}

template <typename T, typename O>
static int linear(const void *x, long long x_st, const LinArgs &a, void *ws, int32_t *status, cudaStream_t s) {
    if (use_few(a.M, a.K)) return launch_few<T, O>(x, x_st, a, s);
    if (!ws) return RESS_E_ARG;
    int8_t *x8 = reinterpret_cast<int8_t *>(ws);
    float *sx = reinterpret_cast<float *>(x8 + ((size_t)a.M * a.K + 255) / 256 * 256);
    const int rc = launch_quant((const T *)x, x_st, a.M, a.K, x8, sx, s);
    if (rc != RESS_OK) return rc;
    const int split = pick_split(a);
    if (split == 4) return launch_split<4, O>(x8, sx, a, status, s);
    if (split == 2) return launch_split<2, O>(x8, sx, a, status, s);
    switch (pick_tile(a)) {
        case 0: return launch_gemm<2, 256, O>(x8, sx, a, status, s);
        case 1: return launch_gemm<1, 128, O>(x8, sx, a, status, s);
        default: return launch_gemm<1, 64, O>(x8, sx, a, status, s);
    }
}

}  // namespace i8
}  // namespace ress

using namespace ress;

extern "C" int ress_int8_quant_rows(const void *x, int dtype, int M, int K, long long x_st, int8_t *x8, float *scale,
                                    ress_stream_t stream) {
    if (!x || !x8 || !scale || M <= 0 || K <= 0 || x_st < K) return RESS_E_ARG;
    if (dtype != RESS_BF16 && dtype != RESS_F32) return RESS_E_DTYPE;
    if (K % 16 != 0 || K > (1 << 17)) return RESS_E_SHAPE;
    const int size = dtype == RESS_BF16 ? 2 : 4;
    if ((((uintptr_t)x | (uintptr_t)x8) & 15) || ((x_st * size) & 15)) return RESS_E_ARG;
    if (dtype == RESS_BF16)
        return i8::launch_quant((const __nv_bfloat16 *)x, x_st, M, K, x8, scale, (cudaStream_t)stream);
    return i8::launch_quant((const float *)x, x_st, M, K, x8, scale, (cudaStream_t)stream);
}

extern "C" size_t ress_int8_linear_workspace(int M, int K) {
    return M > 0 && K > 0 ? i8::workspace(M, K) : 0;
}

extern "C" int ress_int8_linear(const void *x, int dtype, int M, int N, int K, long long x_st, const int8_t *w8,
                                const float *w_scale, const float *bias, int gelu, void *out, int out_dtype,
                                long long out_st, void *workspace, int32_t *status, ress_stream_t stream) {
    if (!x || !w8 || !w_scale || !out || !status || M <= 0 || N <= 0 || K <= 0 || x_st < K || out_st < N)
        return RESS_E_ARG;
    if ((dtype != RESS_BF16 && dtype != RESS_F32) || (out_dtype != RESS_BF16 && out_dtype != RESS_F32))
        return RESS_E_DTYPE;
    if (K % 16 != 0 || K > (1 << 17)) return RESS_E_SHAPE;
    const int size = dtype == RESS_BF16 ? 2 : 4;
    if ((((uintptr_t)x | (uintptr_t)w8) & 15) || ((x_st * size) & 15)) return RESS_E_ARG;
    if (((uintptr_t)workspace & 15) || M > (1 << 26)) return RESS_E_ARG;
    const i8::LinArgs a{w8, w_scale, bias, out, out_st, M, N, K, gelu};
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == RESS_BF16)
        return out_dtype == RESS_BF16 ? i8::linear<__nv_bfloat16, __nv_bfloat16>(x, x_st, a, workspace, status, s)
                                      : i8::linear<__nv_bfloat16, float>(x, x_st, a, workspace, status, s);
    return out_dtype == RESS_BF16 ? i8::linear<float, __nv_bfloat16>(x, x_st, a, workspace, status, s)
                                  : i8::linear<float, float>(x, x_st, a, workspace, status, s);
}

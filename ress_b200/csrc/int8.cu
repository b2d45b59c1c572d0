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
// d: the scale, or 1 where it is 0.  |x / d| rounds to 127 at most (a scale
// among the subnormals can be off by more; the conversion saturates).
__device__ __forceinline__ uint32_t quant4(float a, float b, float c, float e, float d) {
    const int q0 = round_s8(__fdiv_rn(a, d)), q1 = round_s8(__fdiv_rn(b, d));
    const int q2 = round_s8(__fdiv_rn(c, d)), q3 = round_s8(__fdiv_rn(e, d));
    return __byte_perm(__byte_perm(q0, q1, 0x0040), __byte_perm(q2, q3, 0x0040), 0x5410);
}
__device__ __forceinline__ uint32_t amax8(const float (&x)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(x[j]) & 0x7FFFFFFFu);
    return m;
}

__device__ __forceinline__ float finish(int acc, float sx, float sw, float bias, int gelu) {
    float y = __fadd_rn(__fmul_rn(__fmul_rn((float)acc, sx), sw), bias);
    if (gelu) y = 0.5f * y * (1.0f + erff(y * 0.70710678118654752f));
    return y;
}

// Rows to int8 with one scale each: one warp per row, the row read twice
// (the second time from the caches).
constexpr int QUANT_NT = 256;
template <typename T>
__global__ void __launch_bounds__(QUANT_NT) quant_rows_kernel(const T *__restrict__ x, long long x_st, int M, int K,
                                                              int8_t *__restrict__ q, float *__restrict__ scale) {
    const int lane = threadIdx.x & 31;
    const long long m = ((long long)blockIdx.x * QUANT_NT + threadIdx.x) >> 5;
    if (m >= M) return;
    const T *row = x + m * x_st;
    uint32_t am = 0;
    for (int k = lane * 8; k < K; k += 256) {
        float v[8];
        load8(row + k, v);
        am = max(am, amax8(v));
    }
    am = __reduce_max_sync(0xffffffffu, am);
    const float s = row_scale(am), d = s > 0.0f ? s : 1.0f;
    for (int k = lane * 8; k < K; k += 256) {
        float v[8];
        load8(row + k, v);
        *reinterpret_cast<uint2 *>(q + m * K + k) =
            make_uint2(quant4(v[0], v[1], v[2], v[3], d), quant4(v[4], v[5], v[6], v[7], d));
    }
    if (lane == 0) scale[m] = s;
}

// ------------------------------------------------------------------ few rows
// Sixteen tokens a CTA: they are quantised into shared memory by every CTA
// (they are few, and no second launch is needed), each warp then streams
// eight weight rows through mma.sync.m16n8k32 straight from global memory.
// A lane's 16-byte piece of a row serves two k-steps.
constexpr int FEW_NT = 128, FEW_M = 16;
template <typename T, typename O>
__global__ void __launch_bounds__(FEW_NT) few_kernel(const T *__restrict__ x, long long x_st, const LinArgs a) {
    extern __shared__ __align__(16) unsigned char xs[];  // FEW_M rows of Kp + 16 bytes
    __shared__ float sx[FEW_M];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int m0 = blockIdx.y * FEW_M;
    const int Kp = (a.K + 63) & ~63, pitch = Kp + 16;
    for (int r = warp; r < FEW_M; r += FEW_NT / 32) {
        const int m = m0 + r;
        uint32_t am = 0;
        const T *row = x + (long long)m * x_st;
        if (m < a.M)
            for (int k = lane * 8; k < a.K; k += 256) {
                float v[8];
                load8(row + k, v);
                am = max(am, amax8(v));
            }
        am = __reduce_max_sync(0xffffffffu, am);
        const float s = row_scale(am), d = s > 0.0f ? s : 1.0f;
        for (int k = lane * 8; k < Kp; k += 256) {
            uint2 w = make_uint2(0, 0);
            if (m < a.M && k < a.K) {
                float v[8];
                load8(row + k, v);
                w = make_uint2(quant4(v[0], v[1], v[2], v[3], d), quant4(v[4], v[5], v[6], v[7], d));
            }
            *reinterpret_cast<uint2 *>(xs + r * pitch + k) = w;
        }
        if (lane == 0) sx[r] = s;
    }
    __syncthreads();
    const int n0 = (blockIdx.x * (FEW_NT / 32) + warp) * 8;
    if (n0 >= a.N) return;
    const int n = n0 + g;
    const int8_t *wr = a.w + (long long)min(n, a.N - 1) * a.K;
    int c[4] = {};
#pragma unroll 4
    for (int k = t * 16; k < Kp; k += 64) {
        const uint4 b = k < a.K ? __ldg(reinterpret_cast<const uint4 *>(wr + k)) : make_uint4(0, 0, 0, 0);
        const uint4 p = *reinterpret_cast<const uint4 *>(xs + g * pitch + k);
        const uint4 q = *reinterpret_cast<const uint4 *>(xs + (g + 8) * pitch + k);
        asm volatile(
            "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
            : "r"(p.x), "r"(q.x), "r"(p.y), "r"(q.y), "r"(b.x), "r"(b.y));
        asm volatile(
            "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
            : "r"(p.z), "r"(q.z), "r"(p.w), "r"(q.w), "r"(b.z), "r"(b.w));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = g + (i >> 1) * 8, col = n0 + 2 * t + (i & 1);
        if (m0 + r < a.M && col < a.N) {
            const float y = finish(c[i], sx[r], a.w_scale[col], a.bias != nullptr ? a.bias[col] : 0.0f, a.gelu);
            DT<O>::store(reinterpret_cast<O *>(a.out), (size_t)((m0 + r) * a.out_st + col), y);
        }
    }
}

template <typename T, typename O>
static int launch_few(const void *x, long long x_st, const LinArgs &a, cudaStream_t s) {
    const size_t smem = (size_t)FEW_M * (((a.K + 63) & ~63) + 16);
    if (smem > 220 * 1024 || (a.M + FEW_M - 1) / FEW_M > 65535) return RESS_E_SHAPE;
    set_smem_attr((const void *)few_kernel<T, O>, smem);
    const dim3 grid((a.N + 31) / 32, (a.M + FEW_M - 1) / FEW_M);
    few_kernel<T, O><<<grid, FEW_NT, smem, s>>>((const T *)x, x_st, a);
    return cudaGetLastError() == cudaSuccess ? RESS_OK : RESS_E_LAUNCH;
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
    const unsigned blocks = (unsigned)(((long long)M * 32 + i8::QUANT_NT - 1) / i8::QUANT_NT);
    if (dtype == RESS_BF16)
        i8::quant_rows_kernel<<<blocks, i8::QUANT_NT, 0, (cudaStream_t)stream>>>((const __nv_bfloat16 *)x, x_st, M, K, x8,
                                                                                 scale);
    else
        i8::quant_rows_kernel<<<blocks, i8::QUANT_NT, 0, (cudaStream_t)stream>>>((const float *)x, x_st, M, K, x8, scale);
    return cudaGetLastError() == cudaSuccess ? RESS_OK : RESS_E_LAUNCH;
}

extern "C" size_t ress_int8_linear_workspace(int M, int K) {
    (void)M;
    (void)K;
    return 0;
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
    (void)workspace;
    const i8::LinArgs a{w8, w_scale, bias, out, out_st, M, N, K, gelu};
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == RESS_BF16)
        return out_dtype == RESS_BF16 ? i8::launch_few<__nv_bfloat16, __nv_bfloat16>(x, x_st, a, s)
                                      : i8::launch_few<__nv_bfloat16, float>(x, x_st, a, s);
    return out_dtype == RESS_BF16 ? i8::launch_few<float, __nv_bfloat16>(x, x_st, a, s)
                                  : i8::launch_few<float, float>(x, x_st, a, s);
}

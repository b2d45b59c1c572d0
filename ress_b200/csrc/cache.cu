// cache.cu -- new tokens into the paged 8-bit cache: q/k LayerNorm, the 2-D
// rotary embedding and the quantisation in one pass over the projection.
//
// A CTA takes one page of a stream and a few of its heads in turn: 512
// threads, eight per token slot.  Thread i of the eight holds dims d..d+3 and
// d+16..d+19, d = 32*(i/4) + 4*(i%4): the two halves of a rotated pair meet
// in one thread, the eight's loads still cover the row, and cos and sin are
// read once for all heads.  With the page in registers its largest magnitude
// is one reduction away, and codes are written once.  A head's rows are asked
// for while the head before is worked on.  All math is fp32, two lanes an
// instruction: LayerNorm (mean, then mean of squared deviations), the
// rotation x*cos + rotate_half(x)*sin, then
//     e = the least integer with max|y| <= 448 * 2^e,  code = e4m3(y / 2^e)
// over the page's new tokens of that head; a page that holds tokens already
// keeps the larger of its scale and the new one, and its old codes move by
// the power of two between them.  A value that is not finite makes the
// page's scale NaN, so that attention over it shows it.
// Heads vary fastest in the grid: CTAs that run together read whole rows of
// the projection.  q rows of a shared key/value head are taken in turn.
#include "cache.cuh"

namespace ress {
namespace cache {

constexpr int APP_NT = PAGE * 8;

struct AppendArgs {
    const void *q, *k, *v;
    long long q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;  // elements
    void *q_out;  // (B, T, Hq, 64) contiguous
    int T, group;
    const float *qw, *qb, *kw, *kb;
    float eps;
    const long long *pos;
    const void *cos, *sin;
    int rope_len;
    const int32_t *table, *lens, *n_new;
    long long table_stride;
    int table_width, n_pages;
    Pages K, V;
    int32_t *status;
};

// Eight values of a row as loaded: two pieces of four, 16 dims apart.
template <typename T> struct Raw;
template <> struct Raw<__nv_bfloat16> {
    uint2 u[2];
    __device__ __forceinline__ void load(const __nv_bfloat16 *p) {
        u[0] = __ldg(reinterpret_cast<const uint2 *>(p));
        u[1] = __ldg(reinterpret_cast<const uint2 *>(p + 16));
    }
    __device__ __forceinline__ void clear() { u[0] = u[1] = make_uint2(0, 0); }
    __device__ __forceinline__ void get(f32x2 (&x)[4]) const {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[2 * i] = f2_pack(__uint_as_float(u[i].x << 16), __uint_as_float(u[i].x & 0xFFFF0000u));
            x[2 * i + 1] = f2_pack(__uint_as_float(u[i].y << 16), __uint_as_float(u[i].y & 0xFFFF0000u));
        }
    }
};
template <> struct Raw<float> {
    float4 u[2];
    __device__ __forceinline__ void load(const float *p) {
        u[0] = __ldg(reinterpret_cast<const float4 *>(p));
        u[1] = __ldg(reinterpret_cast<const float4 *>(p + 16));
    }
    __device__ __forceinline__ void clear() { u[0] = u[1] = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ __forceinline__ void get(f32x2 (&x)[4]) const {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[2 * i] = f2_pack(u[i].x, u[i].y);
            x[2 * i + 1] = f2_pack(u[i].z, u[i].w);
        }
    }
};
__device__ __forceinline__ void put(__nv_bfloat16 *p, const f32x2 (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float a, b, c, d;
        f2_unpack(x[2 * i], a, b);
        f2_unpack(x[2 * i + 1], c, d);
        const __nv_bfloat162 lo = __floats2bfloat162_rn(a, b), hi = __floats2bfloat162_rn(c, d);
        *reinterpret_cast<uint2 *>(p + 16 * i) =
            make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
    }
}
__device__ __forceinline__ void put(float *p, const f32x2 (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float4 v;
        f2_unpack(x[2 * i], v.x, v.y);
        f2_unpack(x[2 * i + 1], v.z, v.w);
        *reinterpret_cast<float4 *>(p + 16 * i) = v;
    }
}
// four floats of a norm's weight or bias
__device__ __forceinline__ void affine4(const float *p, f32x2 &a, f32x2 &b) {
    const float4 v = __ldg(reinterpret_cast<const float4 *>(p));
    a = f2_pack(v.x, v.y);
    b = f2_pack(v.z, v.w);
}
// the sum of both lanes of x over the eight threads of a row
__device__ __forceinline__ float row_sum(f32x2 x) {
    float a, b;
    f2_unpack(x, a, b);
    a += b;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    return a;
}
__device__ __forceinline__ f32x2 twice(float x) { return f2_pack(x, x); }

// LayerNorm (where w is given) and rotation of a row, unrounded.  All lanes of
// the warp take part.  sn holds sin of dims 16..19 on, and -sin of dims 0..3.
__device__ __forceinline__ void norm_rotate(f32x2 (&x)[4], int d, float eps, const float *w, const float *b, bool rope,
                                            const f32x2 (&cs)[4], const f32x2 (&sn)[4]) {
    if (w != nullptr) {
        const f32x2 mean = twice(-row_sum(f2_add_rn(f2_add_rn(x[0], x[1]), f2_add_rn(x[2], x[3]))) * (1.0f / HD));
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = f2_add_rn(x[i], mean);
        f32x2 sq = f2_mul_rn(x[0], x[0]);
#pragma unroll
        for (int i = 1; i < 4; ++i) sq = f2_fma_rn(x[i], x[i], sq);
        const f32x2 rstd = twice(rsqrtf(fmaf(row_sum(sq), 1.0f / HD, eps)));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f32x2 w0, w1, b0, b1;
            affine4(w + d + 16 * i, w0, w1);
            affine4(b + d + 16 * i, b0, b1);
            x[2 * i] = f2_fma_rn(f2_mul_rn(x[2 * i], rstd), w0, b0);
            x[2 * i + 1] = f2_fma_rn(f2_mul_rn(x[2 * i + 1], rstd), w1, b1);
        }
    }
    if (rope) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const f32x2 lo = x[i], hi = x[2 + i];
            x[i] = f2_fma_rn(lo, cs[i], f2_mul_rn(hi, sn[i]));
            x[2 + i] = f2_fma_rn(hi, cs[2 + i], f2_mul_rn(lo, sn[2 + i]));
        }
    }
}

// The largest magnitude; NaN if there is one.
__device__ __forceinline__ uint32_t amax_bits(const f32x2 (&x)[4]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a, b;
        f2_unpack(x[i], a, b);
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(m), "f"(fabsf(a)));
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(m), "f"(fabsf(b)));
    }
    return __float_as_uint(m) & 0x7FFFFFFFu;
}

// f = 0 (a page of NaN scale) writes zeros whatever x holds, so that no code is ever NaN
__device__ __forceinline__ void store_codes(uint8_t *p, const f32x2 (&x)[4], float f) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float a, b, c, d;
        f2_unpack(f2_mul_rn(x[2 * i], twice(f)), a, b);
        f2_unpack(f2_mul_rn(x[2 * i + 1], twice(f)), c, d);
        *reinterpret_cast<uint32_t *>(p + 16 * i) = f == 0.0f ? 0u : e4m3x4(a, b, c, d);
    }
}
__device__ __noinline__ void move_codes(uint8_t *p, float f) {
    f32x2 x[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t w = *reinterpret_cast<const uint32_t *>(p + 16 * i);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t h = e4m3_to_half2((uint16_t)(w >> (16 * j)));
            const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&h));
            x[2 * i + j] = f2_pack(v.x, v.y);
        }
    }
    store_codes(p, x, f);
}

// heads: of the cache; the CTA takes [blockIdx.x * per, .. + per) of them.
template <typename T>
__global__ void __launch_bounds__(APP_NT, sizeof(T) == 2 ? 2 : 1) append_kernel(const AppendArgs a, int heads, int per) {
    __shared__ uint32_t red[2][2][APP_NT / 32];
    const int b = blockIdx.z;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int slot = threadIdx.x >> 3, i8 = threadIdx.x & 7, d = (i8 >> 2) * 32 + (i8 & 3) * 4;
    const int len_raw = a.lens[b];
    const int len = max(len_raw, 0);
    const int fill = len % PAGE;
    const int t = (int)blockIdx.y * PAGE + slot - fill;  // the new token that falls into this slot
    const int n_new = a.n_new != nullptr ? min(max(a.n_new[b], 0), a.T) : a.T;
    const bool row = t >= 0 && t < a.T;  // there is a q row (written for padding tokens as well)
    const bool fresh = t >= 0 && t < n_new;
    if (blockIdx.y > 0 && (int)blockIdx.y * PAGE - fill >= a.T) return;
    const int h0 = blockIdx.x * per, h1 = min(h0 + per, heads);

    const T *kp = reinterpret_cast<const T *>(a.k) + b * a.k_sb + t * a.k_st + d;
    const T *vp = reinterpret_cast<const T *>(a.v) + b * a.v_sb + t * a.v_st + d;
    const T *qp = reinterpret_cast<const T *>(a.q) + b * a.q_sb + t * a.q_st + d;
    const bool has_q = a.q != nullptr, rope = a.cos != nullptr;
    Raw<T> rk, rv, rq;
    rk.clear();
    rv.clear();
    rq.clear();
    auto ask_kv = [&](int h) {
        if (fresh) {
            rk.load(kp + h * a.k_sh);
            rv.load(vp + h * a.v_sh);
        }
    };
    auto ask_q = [&](int h) {
        if (has_q && row) rq.load(qp + (long long)h * a.group * a.q_sh);
    };
    ask_kv(h0);
    ask_q(h0);
    f32x2 cs[4] = {}, sn[4] = {};
    if (rope && row) {
        const long long pa = a.pos[((long long)b * a.T + t) * 2 + (d >> 5)];
        const int p = (int)(pa < 0 ? 0 : (pa >= a.rope_len ? a.rope_len - 1 : pa));
        Raw<T> rc, rs;
        rc.load(reinterpret_cast<const T *>(a.cos) + (size_t)p * 32 + (d & 31));
        rs.load(reinterpret_cast<const T *>(a.sin) + (size_t)p * 32 + (d & 31));
        rc.get(cs);
        rs.get(sn);
#pragma unroll
        for (int i = 0; i < 2; ++i) sn[i] ^= 0x8000000080000000ull;
    }
    // the page this CTA writes, if any token falls into it
    const long long at = (long long)(len / PAGE) + blockIdx.y;
    const bool any = (int)blockIdx.y * PAGE < fill + n_new && n_new > 0;
    int page = -1;
    if (any && at < a.table_width) page = a.table[b * a.table_stride + at];
    const bool ok = page >= 0 && page < a.n_pages && len_raw >= 0;
    if (any && !ok && threadIdx.x == 0) atomicOr(a.status, RESS_STATUS_CACHE_RANGE);
    const bool held = blockIdx.y == 0 && fill > 0;

    for (int h = h0; h < h1; ++h) {
        f32x2 xk[4], xv[4];
        rk.get(xk);
        const Raw<T> v_now = rv;  // as loaded: half the registers
        if (h + 1 < h1) ask_kv(h + 1);
        norm_rotate(xk, d, a.eps, a.kw, a.kb, rope, cs, sn);
        uint32_t (*r)[APP_NT / 32] = red[h & 1];  // the other one may still be read
        const uint32_t mk = __reduce_max_sync(0xffffffffu, fresh ? amax_bits(xk) : 0u);
        v_now.get(xv);
        const uint32_t mv = __reduce_max_sync(0xffffffffu, fresh ? amax_bits(xv) : 0u);
        if (lane == 0) {
            r[0][warp] = mk;
            r[1][warp] = mv;
        }
        // the scales of a page that holds tokens already, read before anyone writes them
        int old_k = 0, old_v = 0;
        if (ok && held) {
            old_k = a.K.scale[page * a.K.scale_stride + h];
            old_v = a.V.scale[page * a.V.scale_stride + h];
        }
        __syncthreads();
        if (ok) {
            const int uk = max(scale_code(__reduce_max_sync(0xffffffffu, r[0][lane & 15])), old_k);
            const int uv = max(scale_code(__reduce_max_sync(0xffffffffu, r[1][lane & 15])), old_v);
            uint8_t *pk = a.K.codes + page * a.K.page_stride + h * a.K.head_stride + slot * HD + d;
            uint8_t *pv = a.V.codes + page * a.V.page_stride + h * a.V.head_stride + slot * HD + d;
            if (fresh) {
                store_codes(pk, xk, scale_inverse(uk));
                v_now.get(xv);
                store_codes(pv, xv, scale_inverse(uv));
            } else if (held && slot < fill) {
                if (uk != old_k) move_codes(pk, scale_value(old_k) * scale_inverse(uk));
                if (uv != old_v) move_codes(pv, scale_value(old_v) * scale_inverse(uv));
            }
            if (threadIdx.x == 0) {
                a.K.scale[page * a.K.scale_stride + h] = (uint8_t)uk;
                a.V.scale[page * a.V.scale_stride + h] = (uint8_t)uv;
            }
        }
        if (!has_q) continue;
        T *qo = reinterpret_cast<T *>(a.q_out) + (((long long)b * a.T + t) * heads + h) * a.group * HD + d;
        for (int g = 0; g < a.group; ++g) {
            f32x2 xq[4];
            if (g > 0 && row) rq.load(qp + ((long long)h * a.group + g) * a.q_sh);
            rq.get(xq);
            if (g + 1 == a.group && h + 1 < h1) ask_q(h + 1);
            norm_rotate(xq, d, a.eps, a.qw, a.qb, rope, cs, sn);
            if (row) put(qo + (long long)g * HD, xq);
        }
    }
}

}  // namespace cache
}  // namespace ress

using namespace ress;

extern "C" int ress_cache_append(const ress_cache *cache, const ress_append_args *args, int32_t *status,
                                 ress_stream_t stream) {
    const int rc = cache::check_cache(cache);
    if (rc != RESS_OK) return rc;
    if (!args || !status || !args->k || !args->v || args->tokens <= 0) return RESS_E_ARG;
    const ress_append_args &g = *args;
    if ((g.q != nullptr) != (g.q_out != nullptr) || (g.q && (g.q_heads <= 0 || g.q_heads % cache->heads != 0)))
        return RESS_E_ARG;
    if ((g.qn_weight == nullptr) != (g.qn_bias == nullptr) || (g.kn_weight == nullptr) != (g.kn_bias == nullptr))
        return RESS_E_ARG;
    if ((g.rope_cos == nullptr) != (g.rope_sin == nullptr) || (g.rope_cos != nullptr && (!g.pos || g.rope_len <= 0)))
        return RESS_E_ARG;
    if (g.dtype != RESS_BF16 && g.dtype != RESS_F32) return RESS_E_DTYPE;
    // loads of up to 16 bytes
    const int size = g.dtype == RESS_BF16 ? 2 : 4;
    if (((uintptr_t)g.q | (uintptr_t)g.k | (uintptr_t)g.v | (uintptr_t)g.q_out | (uintptr_t)g.rope_cos |
         (uintptr_t)g.rope_sin | (uintptr_t)g.qn_weight | (uintptr_t)g.qn_bias | (uintptr_t)g.kn_weight |
         (uintptr_t)g.kn_bias) & 15)
        return RESS_E_ARG;
    if (((g.k_sb | g.k_st | g.k_sh | g.v_sb | g.v_st | g.v_sh) * size) & 15) return RESS_E_ARG;
    if (g.q && ((g.q_sb | g.q_st | g.q_sh) * size) & 15) return RESS_E_ARG;
    const int64_t pages = (g.tokens + cache::PAGE - 2) / cache::PAGE + 1;  // that the tokens can reach into
    if (pages > 65535 || g.rope_len > (1 << 30) || g.q_heads > (1 << 20)) return RESS_E_SHAPE;
    cache::AppendArgs a;
    a.q = g.q; a.k = g.k; a.v = g.v;
    a.q_sb = g.q_sb; a.q_st = g.q_st; a.q_sh = g.q_sh;
    a.k_sb = g.k_sb; a.k_st = g.k_st; a.k_sh = g.k_sh;
    a.v_sb = g.v_sb; a.v_st = g.v_st; a.v_sh = g.v_sh;
    a.q_out = g.q_out;
    a.T = (int)g.tokens;
    a.group = g.q ? (int)(g.q_heads / cache->heads) : 0;
    a.qw = g.qn_weight; a.qb = g.qn_bias; a.kw = g.kn_weight; a.kb = g.kn_bias;
    a.eps = (float)g.eps;
    a.pos = reinterpret_cast<const long long *>(g.pos);
    a.cos = g.rope_cos; a.sin = g.rope_sin; a.rope_len = (int)g.rope_len;
    a.table = cache->table; a.lens = cache->lens; a.n_new = g.n_new;
    a.table_stride = cache->table_stride; a.table_width = (int)cache->table_width; a.n_pages = (int)cache->n_pages;
    a.K = {cache->k_pages, cache->k_scale, cache->page_stride, cache->head_stride, cache->scale_stride};
    a.V = {cache->v_pages, cache->v_scale, cache->page_stride, cache->head_stride, cache->scale_stride};
    a.status = status;
    // heads a CTA takes in turn: one while the CTAs fit on the GPU at once
    // (two per SM), up to four beyond that, where it hides a head's loads
    const int64_t ctas = cache->heads * pages * cache->streams;
    int per = 1;
    while (per < 4 && ctas / (2 * per) >= 2 * 148) per *= 2;
    const int heads = (int)cache->heads;
    const dim3 grid((unsigned)((heads + per - 1) / per), (unsigned)pages, (unsigned)cache->streams);
    if (g.dtype == RESS_BF16)
        cache::append_kernel<__nv_bfloat16><<<grid, cache::APP_NT, 0, (cudaStream_t)stream>>>(a, heads, per);
    else
        cache::append_kernel<float><<<grid, cache::APP_NT, 0, (cudaStream_t)stream>>>(a, heads, per);
    return cudaGetLastError() == cudaSuccess ? RESS_OK : RESS_E_LAUNCH;
}

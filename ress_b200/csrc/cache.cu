// cache.cu -- new tokens into the paged 8-bit cache: q/k LayerNorm, the 2-D
// rotary embedding and the quantisation in one pass over the projection.
//
// A CTA takes one page of a stream and a few of its heads in turn: 256
// threads, eight per token, two tokens a thread.  Thread i of the eight holds
// dims d..d+3 and d+16..d+19, d = 32*(i/4) + 4*(i%4): the two halves of a
// rotated pair meet in one thread, the eight's loads still cover the row, and
// cos and sin are read once for all heads.  With the page in registers its
// largest magnitude is one reduction away, and codes are written once.  A
// head's rows are asked for while the head before is worked on.  All math is
// fp32, two lanes an instruction: LayerNorm (mean, then mean of squared
// deviations), the rotation x*cos + rotate_half(x)*sin, then
//     e = the least integer with max|y| <= 448 * 2^e,  code = e4m3(y / 2^e)
// over the page's new tokens of that head; a page that holds tokens already
// keeps the larger of its scale and the new one, and its old codes move by
// the power of two between them.  A value that is not finite makes the
// page's scale NaN, so that attention over it shows it.
// Heads vary fastest in the grid: CTAs that run together read whole rows of
// the projection.  q rows of a shared key/value head are taken in turn.
//
// 43,968 tokens of 16 heads, bf16, with norms and rotation: 450 MB, 115 us, 3.9
// TB/s of the 6.45 that a copy reaches; what bounds it is the L1's loads and the
// instructions issued.  The norms' weights are a third of the loads, which two
// tokens a thread share: with one token a thread 156 us (at twice the warps),
// with four 151 (spilling).  A single token 3.5 us, 24 streams of five 4.9, a
// frame of 1374 tokens 7.9, each close to a launch and two memory latencies.
#include "cache.cuh"

namespace ress {
namespace cache {

constexpr int ROWS = 2;  // of a thread, PAGE / ROWS slots apart
constexpr int APP_NT = PAGE / ROWS * 8;

struct AppendArgs {
    const void *q, *k, *v;
    long long q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;  // elements
    void *q_out;  // (B, T, Hq, 64) contiguous
    int T, group;
    const void *qw, *qb, *kw, *kb;
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
// four values of a norm's weight or bias
__device__ __forceinline__ void affine4(const float *p, f32x2 &a, f32x2 &b) {
    const float4 v = __ldg(reinterpret_cast<const float4 *>(p));
    a = f2_pack(v.x, v.y);
    b = f2_pack(v.z, v.w);
}
__device__ __forceinline__ void affine4(const __nv_bfloat16 *p, f32x2 &a, f32x2 &b) {
    const uint2 u = __ldg(reinterpret_cast<const uint2 *>(p));
    a = f2_pack(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u));
    b = f2_pack(__uint_as_float(u.y << 16), __uint_as_float(u.y & 0xFFFF0000u));
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

// LayerNorm (where w is given) and rotation of a thread's rows, unrounded.  All
// lanes of the warp take part.  sn holds sin of dims 16..19 on, and -sin of
// dims 0..3.
template <typename W>
__device__ __forceinline__ void norm_rotate(f32x2 (&x)[ROWS][4], int d, float eps, const W *w, const W *b, bool rope,
                                            const f32x2 (&cs)[ROWS][4], const f32x2 (&sn)[ROWS][4]) {
    if (w != nullptr) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const f32x2 mean =
                twice(-row_sum(f2_add_rn(f2_add_rn(x[r][0], x[r][1]), f2_add_rn(x[r][2], x[r][3]))) * (1.0f / HD));
#pragma unroll
            for (int i = 0; i < 4; ++i) x[r][i] = f2_add_rn(x[r][i], mean);
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            f32x2 sq = f2_mul_rn(x[r][0], x[r][0]);
#pragma unroll
            for (int i = 1; i < 4; ++i) sq = f2_fma_rn(x[r][i], x[r][i], sq);
            const f32x2 rstd = twice(rsqrtf(fmaf(row_sum(sq), 1.0f / HD, eps)));
#pragma unroll
            for (int i = 0; i < 4; ++i) x[r][i] = f2_mul_rn(x[r][i], rstd);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f32x2 w0, w1, b0, b1;
            affine4(w + d + 16 * i, w0, w1);
            affine4(b + d + 16 * i, b0, b1);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                x[r][2 * i] = f2_fma_rn(x[r][2 * i], w0, b0);
                x[r][2 * i + 1] = f2_fma_rn(x[r][2 * i + 1], w1, b1);
            }
        }
    }
    if (rope) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const f32x2 lo = x[r][i], hi = x[r][2 + i];
                x[r][i] = f2_fma_rn(lo, cs[r][i], f2_mul_rn(hi, sn[r][i]));
                x[r][2 + i] = f2_fma_rn(hi, cs[r][2 + i], f2_mul_rn(lo, sn[r][2 + i]));
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

// T, W: types of the rows and of the norms.
// heads: of the cache; the CTA takes [blockIdx.x * per, .. + per) of them.
template <typename T, typename W>
__global__ void __launch_bounds__(APP_NT, 2) append_kernel(const AppendArgs a, int heads, int per) {
    constexpr int WARPS = APP_NT / 32;
    __shared__ uint32_t red[2][2][WARPS];
    const int b = blockIdx.z;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int slot = threadIdx.x >> 3, i8 = threadIdx.x & 7, d = (i8 >> 2) * 32 + (i8 & 3) * 4;
    const int len_raw = a.lens[b];
    const int len = max(len_raw, 0);
    const int fill = len % PAGE;
    const int n_new = a.n_new != nullptr ? min(max(a.n_new[b], 0), a.T) : a.T;
    if (blockIdx.y > 0 && (int)blockIdx.y * PAGE - fill >= a.T) return;
    const int h0 = blockIdx.x * per, h1 = min(h0 + per, heads);
    // the new token that falls into the thread's first slot; the others follow
    // PAGE / ROWS tokens apart
    const int t0 = (int)blockIdx.y * PAGE + slot - fill;
    bool row[ROWS], fresh[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const int t = t0 + r * (PAGE / ROWS);
        row[r] = t >= 0 && t < a.T;  // there is a q row (written for padding tokens as well)
        fresh[r] = t >= 0 && t < n_new;
    }

    const T *kp = reinterpret_cast<const T *>(a.k) + b * a.k_sb + t0 * a.k_st + d;
    const T *vp = reinterpret_cast<const T *>(a.v) + b * a.v_sb + t0 * a.v_st + d;
    const T *qp = reinterpret_cast<const T *>(a.q) + b * a.q_sb + t0 * a.q_st + d;
    const W *const qw = reinterpret_cast<const W *>(a.qw), *const qb = reinterpret_cast<const W *>(a.qb);
    const W *const kw = reinterpret_cast<const W *>(a.kw), *const kb = reinterpret_cast<const W *>(a.kb);
    const bool has_q = a.q != nullptr, rope = a.cos != nullptr;
    Raw<T> rk[ROWS], rv[ROWS], rq[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        rk[r].clear();
        rv[r].clear();
        rq[r].clear();
    }
    auto ask_k = [&](int h) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
            if (fresh[r]) rk[r].load(kp + r * (PAGE / ROWS) * a.k_st + h * a.k_sh);
    };
    auto ask_v = [&](int h) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
            if (fresh[r]) rv[r].load(vp + r * (PAGE / ROWS) * a.v_st + h * a.v_sh);
    };
    auto ask_q = [&](long long h) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
            if (has_q && row[r]) rq[r].load(qp + r * (PAGE / ROWS) * a.q_st + h * a.q_sh);
    };
    // fp32 rows leave no registers to ask for a head's v and q a head ahead
    constexpr bool AHEAD = sizeof(T) == 2;
    ask_k(h0);
    ask_v(h0);
    if (AHEAD) ask_q((long long)h0 * a.group);
    f32x2 cs[ROWS][4] = {}, sn[ROWS][4] = {};
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
        if (rope && row[r]) {
            const long long pa = a.pos[((long long)b * a.T + t0 + r * (PAGE / ROWS)) * 2 + (d >> 5)];
            const int p = (int)(pa < 0 ? 0 : (pa >= a.rope_len ? a.rope_len - 1 : pa));
            Raw<T> rc, rs;
            rc.load(reinterpret_cast<const T *>(a.cos) + (size_t)p * 32 + (d & 31));
            rs.load(reinterpret_cast<const T *>(a.sin) + (size_t)p * 32 + (d & 31));
            rc.get(cs[r]);
            rs.get(sn[r]);
#pragma unroll
            for (int i = 0; i < 2; ++i) sn[r][i] ^= 0x8000000080000000ull;
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
        f32x2 x[ROWS][4];
        Raw<T> v_now[ROWS];  // as loaded: half the registers
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            rk[r].get(x[r]);
            v_now[r] = rv[r];
        }
        if (h + 1 < h1) {
            ask_k(h + 1);
            if (AHEAD) ask_v(h + 1);
        }
        norm_rotate(x, d, a.eps, kw, kb, rope, cs, sn);
        uint32_t (*red_h)[WARPS] = red[h & 1];  // the other one may still be read
        uint32_t mk = 0, mv = 0;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            f32x2 xv[4];
            v_now[r].get(xv);
            mk = max(mk, fresh[r] ? amax_bits(x[r]) : 0u);
            mv = max(mv, fresh[r] ? amax_bits(xv) : 0u);
        }
        mk = __reduce_max_sync(0xffffffffu, mk);
        mv = __reduce_max_sync(0xffffffffu, mv);
        if (lane == 0) {
            red_h[0][warp] = mk;
            red_h[1][warp] = mv;
        }
        // the scales of a page that holds tokens already, read before anyone writes them
        int old_k = 0, old_v = 0;
        if (ok && held) {
            old_k = a.K.scale[page * a.K.scale_stride + h];
            old_v = a.V.scale[page * a.V.scale_stride + h];
        }
        __syncthreads();
        if (ok) {
            const int uk = max(scale_code(__reduce_max_sync(0xffffffffu, red_h[0][lane % WARPS])), old_k);
            const int uv = max(scale_code(__reduce_max_sync(0xffffffffu, red_h[1][lane % WARPS])), old_v);
            uint8_t *pk = a.K.codes + page * a.K.page_stride + h * a.K.head_stride + slot * HD + d;
            uint8_t *pv = a.V.codes + page * a.V.page_stride + h * a.V.head_stride + slot * HD + d;
#pragma unroll
            for (int r = 0; r < ROWS; ++r, pk += PAGE / ROWS * HD, pv += PAGE / ROWS * HD) {
                if (fresh[r]) {
                    f32x2 xv[4];
                    store_codes(pk, x[r], scale_inverse(uk));
                    v_now[r].get(xv);
                    store_codes(pv, xv, scale_inverse(uv));
                } else if (held && slot + r * (PAGE / ROWS) < fill) {
                    if (uk != old_k) move_codes(pk, scale_value(old_k) * scale_inverse(uk));
                    if (uv != old_v) move_codes(pv, scale_value(old_v) * scale_inverse(uv));
                }
            }
            if (threadIdx.x == 0) {
                a.K.scale[page * a.K.scale_stride + h] = (uint8_t)uk;
                a.V.scale[page * a.V.scale_stride + h] = (uint8_t)uv;
            }
        }
        if (!AHEAD && h + 1 < h1) ask_v(h + 1);
        if (!has_q) continue;
        const long long q_row = (long long)heads * a.group * HD;
        T *qo = reinterpret_cast<T *>(a.q_out) + ((long long)b * a.T + t0) * q_row + (long long)h * a.group * HD + d;
        for (int g = 0; g < a.group; ++g, qo += HD) {
            if (!AHEAD || g > 0) ask_q((long long)h * a.group + g);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) rq[r].get(x[r]);
            if (AHEAD && g + 1 == a.group && h + 1 < h1) ask_q((long long)(h + 1) * a.group);
            norm_rotate(x, d, a.eps, qw, qb, rope, cs, sn);
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
                if (row[r]) put(qo + r * (PAGE / ROWS) * q_row, x[r]);
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
    const bool bf16 = (g.dtype & ~(int64_t)RESS_BF16_NORMS) == RESS_BF16, bf16_norms = (g.dtype & RESS_BF16_NORMS) != 0;
    if (!bf16 && g.dtype != RESS_F32) return RESS_E_DTYPE;
    // loads of up to 16 bytes
    const int size = bf16 ? 2 : 4;
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
    // Heads a CTA takes in turn (a head's loads are hidden behind the head
    // before): the count whose waves of two CTAs per SM take least, where a q row
    // costs about a third of a head's k and v and a CTA's start nearly as much as
    // they do.  Measured, us at 1, 2, 4, 8 heads: 43,968 tokens of 16 heads 146,
    // 119, 110, 107; 10,992 44, 38, 37, 41; 64 streams of one token 13.4, 11.9,
    // 11.9, 11.9; 8 streams of 1374, 16 q heads on 4 20.4, 22.6, 23.6.
    const int64_t ctas = cache->heads * ((g.tokens + cache::PAGE - 1) / cache::PAGE) * cache->streams;
    const int64_t head = 20 + 10 * (int64_t)a.group, start = 27;
    int per = 1;
    int64_t least = INT64_MAX;
    for (int p = 1; p <= 8 && p < 2 * cache->heads; p *= 2) {
        const int64_t cost = ((ctas + p - 1) / p + 2 * 148 - 1) / (2 * 148) * (head * p + start);
        if (cost < least) {
            least = cost;
            per = p;
        }
    }
    const int heads = (int)cache->heads;
    const dim3 grid((unsigned)((heads + per - 1) / per), (unsigned)pages, (unsigned)cache->streams);
    auto kern = !bf16        ? cache::append_kernel<float, float>
                : bf16_norms ? cache::append_kernel<__nv_bfloat16, __nv_bfloat16>
                             : cache::append_kernel<__nv_bfloat16, float>;
    kern<<<grid, cache::APP_NT, 0, (cudaStream_t)stream>>>(a, heads, per);
    return cudaGetLastError() == cudaSuccess ? RESS_OK : RESS_E_LAUNCH;
}

// cache.cu -- new tokens into the paged 8-bit cache: q/k LayerNorm, the 2-D
// rotary embedding and the quantisation in one pass over the projection.
//
// One CTA per (page, key/value head, stream): 512 threads, eight per token
// slot, so that a thread holds eight head dims of one token's k, v and q
// (16-byte bf16 loads, all in flight before the first use).  With the page
// in registers its largest magnitude is one reduction away, and codes are
// written once.  All math is fp32: LayerNorm (mean, then mean of squared
// deviations), the rotation x*cos + rotate_half(x)*sin, then
//     e = the least integer with max|y| <= 448 * 2^e,  code = e4m3(y / 2^e)
// over the page's new tokens of that head; a page that holds tokens already
// keeps the larger of its scale and the new one, and its old codes move by
// the power of two between them.  A value that is not finite makes the
// page's scale NaN, so that attention over it shows it.
// Heads vary fastest in the grid: CTAs that run together read whole rows of
// the projection.  q rows of a shared key/value head are taken in turn.
#include "cache.cuh"
#include "prologue.cuh"

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

// LayerNorm (where w is given) and rotation of one row spread over eight
// lanes, unrounded fp32 in and out.  All lanes of the warp take part.
__device__ __forceinline__ void norm_rotate8(float (&x)[8], int c, float eps, const float *w, const float *b, bool rope,
                                             const float (&cs)[8], const float (&sn)[8]) {
    if (w != nullptr) {
        prologue_row8<float>(x, c, eps, w, b, rope, cs, sn);
    } else if (rope) {
        const bool first = (c & 31) < 16;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float z = __shfl_xor_sync(0xffffffffu, x[j], 2);  // feature j +- 16
            x[j] = __fadd_rn(__fmul_rn(x[j], cs[j]), __fmul_rn(first ? -z : z, sn[j]));
        }
    }
}

__device__ __forceinline__ uint32_t amax8(const float (&x)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(x[j]) & 0x7FFFFFFFu);  // NaN and infinity sort last
    return m;
}

// f = 0 (a page of NaN scale) writes zeros whatever x holds, so that no code is ever NaN
__device__ __forceinline__ void store_codes(uint8_t *dst, const float (&x)[8], float f) {
    if (f == 0.0f) {
        *reinterpret_cast<uint2 *>(dst) = make_uint2(0, 0);
        return;
    }
    const uint32_t lo = e4m3x4(x[0] * f, x[1] * f, x[2] * f, x[3] * f);
    const uint32_t hi = e4m3x4(x[4] * f, x[5] * f, x[6] * f, x[7] * f);
    *reinterpret_cast<uint2 *>(dst) = make_uint2(lo, hi);
}

__device__ __forceinline__ void move_codes(uint8_t *p, float f) {
    const uint2 old = *reinterpret_cast<const uint2 *>(p);
    float x[8];
    const uint32_t w[2] = {old.x, old.y};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t h = e4m3_to_half2((uint16_t)(w[j >> 1] >> ((j & 1) * 16)));
        const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&h));
        x[2 * j] = v.x;
        x[2 * j + 1] = v.y;
    }
    store_codes(p, x, f);
}

template <typename T>
__global__ void __launch_bounds__(APP_NT) append_kernel(const AppendArgs a) {
    __shared__ uint32_t red[2][APP_NT / 32];
    const int h = blockIdx.x, b = blockIdx.z;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int slot = threadIdx.x >> 3, c = (threadIdx.x & 7) * 8;
    const int len_raw = a.lens[b];
    const int len = max(len_raw, 0);
    const int fill = len % PAGE;
    const int t = (int)blockIdx.y * PAGE + slot - fill;  // the new token that falls into this slot
    const int n_new = a.n_new != nullptr ? min(max(a.n_new[b], 0), a.T) : a.T;
    const bool row = t >= 0 && t < a.T;  // there is a q row (written for padding tokens as well)
    const bool fresh = t >= 0 && t < n_new;
    if (blockIdx.y > 0 && (int)blockIdx.y * PAGE - fill >= a.T) return;

    float xk[8] = {}, xv[8] = {}, xq[8] = {}, cs[8] = {}, sn[8] = {};
    const bool rope = a.cos != nullptr;
    if (fresh) {
        load8(reinterpret_cast<const T *>(a.k) + b * a.k_sb + t * a.k_st + h * a.k_sh + c, xk);
        load8(reinterpret_cast<const T *>(a.v) + b * a.v_sb + t * a.v_st + h * a.v_sh + c, xv);
    }
    const T *qp = reinterpret_cast<const T *>(a.q) + b * a.q_sb + t * a.q_st + (long long)h * a.group * a.q_sh + c;
    const bool has_q = a.q != nullptr;
    if (has_q && row) load8(qp, xq);
    if (rope && row) {
        const long long pa = a.pos[((long long)b * a.T + t) * 2 + (c >> 5)];
        const int p = (int)(pa < 0 ? 0 : (pa >= a.rope_len ? a.rope_len - 1 : pa));
        load8(reinterpret_cast<const T *>(a.cos) + (size_t)p * 32 + (c & 31), cs);
        load8(reinterpret_cast<const T *>(a.sin) + (size_t)p * 32 + (c & 31), sn);
    }
    // the page this CTA writes, if any token falls into it
    const long long at = (long long)(len / PAGE) + blockIdx.y;
    const bool any = (int)blockIdx.y * PAGE < fill + n_new && n_new > 0;
    int page = -1;
    if (any && at < a.table_width) page = a.table[b * a.table_stride + at];
    const bool ok = page >= 0 && page < a.n_pages && len_raw >= 0;
    if (any && !ok && threadIdx.x == 0) atomicOr(a.status, RESS_STATUS_CACHE_RANGE);

    norm_rotate8(xk, c, a.eps, a.kw, a.kb, rope, cs, sn);
    if (!fresh) {
#pragma unroll
        for (int j = 0; j < 8; ++j) xk[j] = 0.0f;
    }
    const uint32_t mk = __reduce_max_sync(0xffffffffu, amax8(xk)), mv = __reduce_max_sync(0xffffffffu, amax8(xv));
    if (lane == 0) {
        red[0][warp] = mk;
        red[1][warp] = mv;
    }
    // the scales of a page that holds tokens already, read before anyone writes them
    const bool held = blockIdx.y == 0 && fill > 0;
    int old_k = 0, old_v = 0;
    if (ok && held) {
        old_k = a.K.scale[page * a.K.scale_stride + h];
        old_v = a.V.scale[page * a.V.scale_stride + h];
    }
    __syncthreads();
    if (ok) {
        const uint32_t rk = __reduce_max_sync(0xffffffffu, red[0][lane & 15]);
        const uint32_t rv = __reduce_max_sync(0xffffffffu, red[1][lane & 15]);
        const int uk = max(scale_code(rk), old_k), uv = max(scale_code(rv), old_v);
        uint8_t *pk = a.K.codes + page * a.K.page_stride + h * a.K.head_stride + slot * HD + c;
        uint8_t *pv = a.V.codes + page * a.V.page_stride + h * a.V.head_stride + slot * HD + c;
        if (fresh) {
            store_codes(pk, xk, scale_inverse(uk));
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
    if (!has_q) return;
    T *qo = reinterpret_cast<T *>(a.q_out) + (((long long)b * a.T + t) * gridDim.x + h) * a.group * HD + c;
    for (int g = 0; g < a.group; ++g) {
        if (g > 0 && row) load8(qp + g * a.q_sh, xq);
        norm_rotate8(xq, c, a.eps, a.qw, a.qb, rope, cs, sn);
        if (row) store8(qo + (long long)g * HD, xq);
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
    // 16-byte loads of eight elements
    const int size = g.dtype == RESS_BF16 ? 2 : 4;
    if (((uintptr_t)g.q | (uintptr_t)g.k | (uintptr_t)g.v | (uintptr_t)g.q_out | (uintptr_t)g.rope_cos |
         (uintptr_t)g.rope_sin) & 15)
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
    const dim3 grid((unsigned)cache->heads, (unsigned)pages, (unsigned)cache->streams);
    if (g.dtype == RESS_BF16)
        cache::append_kernel<__nv_bfloat16><<<grid, cache::APP_NT, 0, (cudaStream_t)stream>>>(a);
    else
        cache::append_kernel<float><<<grid, cache::APP_NT, 0, (cudaStream_t)stream>>>(a);
    return cudaGetLastError() == cudaSuccess ? RESS_OK : RESS_E_LAUNCH;
}

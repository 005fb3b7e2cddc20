// Attention of one new token per row over a paged key-value cache.
//
//     o = sum_t p_t v_t / sum_t p_t,   p_t = exp(scale * q . k_t - m),   m the running maximum
//
// One pass over the row's keys and values; the sums are rescaled when the maximum grows.  All arithmetic in FP32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "kv_place.h"
#include "pdl.cuh"
#include "te_internal.h"

namespace te {

namespace {

struct AttnParams {
    const float* q;
    float* o;
    float* lse;
    const void* kc;
    const void* vc;
    const float* k_scale;
    const float* v_scale;
    const int64_t* page_table;
    const int64_t* lens;
    int64_t qs[2], os[2], kcs[3], vcs[3], ss[3];
    int64_t table_stride, max_pages, pages, window;
    int64_t rows;
    FastDivisor page_size;
    int q_heads, group, d;
    float scale;
    int* status;
};

template <int DTYPE>
__device__ __forceinline__ float stored_value(const void* base, int64_t at) {
    if constexpr (DTYPE == TE_KV_F32) return static_cast<const float*>(base)[at];
    else if constexpr (DTYPE == TE_KV_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[at]);
    else return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<const __nv_fp8_storage_t*>(base)[at], __NV_E4M3)));
}

// One warp per (row, query head), lanes along d.
template <int DTYPE>
__global__ void __launch_bounds__(32) paged_attention_kernel(const AttnParams p) {
    griddep_wait();
    const int lane = threadIdx.x;
    const int64_t r = blockIdx.x / p.q_heads;
    const int h = (int)(blockIdx.x - r * p.q_heads), kh = h / p.group;
    int64_t n = p.lens[r];
    const int64_t most = p.max_pages * (int64_t)p.page_size.divisor;
    if (n > most) {
        n = most;
        if (lane == 0) atomicCAS(p.status, 0, STATUS_BAD_CACHE_PLACE);
    }
    const int64_t first = p.window > 0 && n > p.window ? n - p.window : 0;
    const PageRow table = {p.page_table + r * p.table_stride, p.max_pages, p.pages};
    float q[8], acc[8];
    const int per = (p.d + 31) / 32;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = lane + 32 * i;
        q[i] = i < per && c < p.d ? p.q[r * p.qs[0] + h * p.qs[1] + c] * p.scale : 0.0f;
        acc[i] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int64_t t = first; t < n; ++t) {
        int64_t page;
        uint32_t slot;
        if (!kv_place(table, p.page_size, t, page, slot)) {
            if (lane == 0) atomicCAS(p.status, 0, STATUS_BAD_CACHE_PLACE);
            continue;
        }
        const int64_t ka = page * p.kcs[0] + kh * p.kcs[1] + slot * p.kcs[2], va = page * p.vcs[0] + kh * p.vcs[1] + slot * p.vcs[2];
        float sk = 1.0f, sv = 1.0f;
        if constexpr (DTYPE == TE_KV_E4M3) {
            const int64_t s = page * p.ss[0] + kh * p.ss[1] + slot * p.ss[2];
            sk = p.k_scale[s];
            sv = p.v_scale[s];
        }
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = lane + 32 * i;
            if (i < per && c < p.d) s += q[i] * stored_value<DTYPE>(p.kc, ka + c);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        s *= sk;
        const float top = fmaxf(m, s);
        const float keep = m == top ? 1.0f : expf(m - top), w = s == top ? 1.0f : expf(s - top);
        m = top;
        l = l * keep + w;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = lane + 32 * i;
            if (i < per && c < p.d) acc[i] = acc[i] * keep + w * (sv * stored_value<DTYPE>(p.vc, va + c));
        }
    }
    const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = lane + 32 * i;
        if (i < per && c < p.d) p.o[r * p.os[0] + h * p.os[1] + c] = acc[i] * inv;
    }
    if (p.lse && lane == 0) p.lse[r * p.q_heads + h] = l == 0.0f ? -INFINITY : m + logf(l);
}

int check_desc(const te_paged_attn_desc* t) {
    if (!t || t->rows < 0 || t->q_heads < 0 || t->max_pages < 0) return fail(TE_ERR_BAD_ARGUMENT, "paged attention: bad extents");
    if (int bad = check_kv_cache(t->cache, "paged attention")) return bad;
    const te_kv_cache& c = t->cache;
    if (t->q_heads > 0 && (c.heads == 0 || t->q_heads % c.heads)) return fail(TE_ERR_BAD_ARGUMENT, "paged attention: q_heads must be a multiple of the cache's heads");
    if (t->max_pages > 0 && c.page_size > INT32_MAX / t->max_pages) return fail(TE_ERR_BAD_ARGUMENT, "paged attention: the page table reaches beyond 2^31-1 positions");
    if (t->q_heads > 65535 || (t->q_heads > 0 && t->rows > INT32_MAX / t->q_heads)) return fail(TE_ERR_BAD_ARGUMENT, "paged attention: too many rows or heads");
    if (t->window < 0) return fail(TE_ERR_BAD_ARGUMENT, "paged attention: negative window");
    if (!isfinite(t->scale)) return fail(TE_ERR_BAD_ARGUMENT, "paged attention: scale must be finite");
    if (t->rows == 0 || t->q_heads == 0) return TE_OK;
    if (!t->q || !t->o || !t->lens || (t->max_pages > 0 && !t->page_table)) return fail(TE_ERR_BAD_ARGUMENT, "paged attention: NULL pointer");
    if (t->page_table_stride < 0 || t->q_strides[0] < 0 || t->q_strides[1] < 0 || t->o_strides[0] < 0 || t->o_strides[1] < 0)
        return fail(TE_ERR_BAD_ARGUMENT, "paged attention: negative stride");
    if ((t->rows > 1 && t->o_strides[0] < c.d) || (t->q_heads > 1 && t->o_strides[1] < c.d))
        return fail(TE_ERR_UNSUPPORTED_LAYOUT, "paged attention: heads of the output overlap");
    return TE_OK;
}

}  // namespace

}  // namespace te

using namespace te;

extern "C" {

int te_b200_paged_attention_workspace_size(const te_paged_attn_desc* d, int sm_count, size_t* out_bytes) {
    if (!out_bytes || sm_count < 1) return fail(TE_ERR_BAD_ARGUMENT, "paged attention: out_bytes is NULL or sm_count not positive");
    if (int bad = check_desc(d)) return bad;
    *out_bytes = 0;
    return TE_OK;
}

int te_b200_paged_attention(te_b200_ctx* ctx, const te_paged_attn_desc* t, te_stream_t stream) {
    if (int bad = check_desc(t)) return bad;
    if (int bad = check_ctx(ctx)) return bad;
    if (t->rows == 0 || t->q_heads == 0) return TE_OK;
    const te_kv_cache& c = t->cache;
    AttnParams p;
    p.q = t->q; p.o = t->o; p.lse = t->lse; p.kc = c.k; p.vc = c.v; p.k_scale = c.k_scale; p.v_scale = c.v_scale;
    p.page_table = t->page_table; p.lens = t->lens;
    for (int i = 0; i < 2; ++i) { p.qs[i] = t->q_strides[i]; p.os[i] = t->o_strides[i]; }
    for (int i = 0; i < 3; ++i) { p.kcs[i] = c.k_strides[i]; p.vcs[i] = c.v_strides[i]; p.ss[i] = c.scale_strides[i]; }
    p.table_stride = t->page_table_stride; p.max_pages = t->max_pages; p.pages = c.pages; p.window = t->window;
    p.rows = t->rows;
    p.page_size = make_fast_divisor((uint32_t)c.page_size);
    p.q_heads = (int)t->q_heads; p.group = (int)(t->q_heads / c.heads); p.d = (int)c.d;
    p.scale = t->scale;
    p.status = ctx->d_status;
    const dim3 grid((unsigned)(t->rows * t->q_heads)), block(32);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (c.dtype == TE_KV_F32) e = launch_pdl(paged_attention_kernel<TE_KV_F32>, grid, block, 0, st, p);
    else if (c.dtype == TE_KV_BF16) e = launch_pdl(paged_attention_kernel<TE_KV_BF16>, grid, block, 0, st, p);
    else e = launch_pdl(paged_attention_kernel<TE_KV_E4M3>, grid, block, 0, st, p);
    if (e != cudaSuccess) return cuda_fail(e, "paged_attention_kernel launch");
    ctx->launches += 1;
    return TE_OK;
}

}  // extern "C"

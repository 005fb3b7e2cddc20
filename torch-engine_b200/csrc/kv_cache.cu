// The paged key-value cache: tokens written into it (rounded to the cache's type, 8-bit rows with a power-of-two scale of
// their own) and read back as FP32.  Both directions are streaming kernels bound by HBM: 4 B of FP32 and 4, 2 or 1 B of
// cache per element (and 4 B of scale per 8-bit row).
//
// A row is the d elements of one (token, head) of k or of v.  A group of LANES lanes holds it, four elements a lane (eight
// for d > 128), so that FP32 moves in float4s, the largest magnitude of a row is one butterfly within the group, and a
// row's bytes leave in one coalesced store.  Consecutive groups take consecutive tokens of one head, which lie side by side
// in the cache's usual order [pages, heads, page_size, d].
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kv_place.h"
#include "pdl.cuh"
#include "te_internal.h"

namespace te {

namespace {

struct KvParams {
    float* k;
    float* v;
    void* kc;
    void* vc;
    float* k_scale;
    float* v_scale;
    const int64_t* page_table;
    const int64_t* positions;
    int64_t ks[3], vs[3], ps[2], kcs[3], vcs[3], ss[3];
    int64_t table_stride, max_pages, pages;
    int64_t rows;               // B * H * T, T fastest
    FastDivisor page_size;
    int T, H, d;
    int* status;
};

template <int DTYPE> struct Stored;
template <> struct Stored<TE_KV_F32> { typedef float type; };
template <> struct Stored<TE_KV_BF16> { typedef __nv_bfloat16 type; };
template <> struct Stored<TE_KV_E4M3> { typedef unsigned char type; };

__device__ __forceinline__ bool is_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }   // -126 <= e <= 127

// The exponent of the smallest 2^e, e >= -126, with amax <= 448 * 2^e = 1.75 * 2^(e + 8).
__device__ __forceinline__ int scale_exponent(float amax) {
    const unsigned bits = __float_as_uint(amax);
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < -126 ? -126 : e;
}

template <bool VEC>
__device__ __forceinline__ float4 load4(const float* p) {
    if constexpr (VEC) return *reinterpret_cast<const float4*>(p);
    else return make_float4(p[0], p[1], p[2], p[3]);
}
template <bool VEC>
__device__ __forceinline__ void store4(float* p, float4 x) {
    if constexpr (VEC) *reinterpret_cast<float4*>(p) = x;
    else { p[0] = x.x; p[1] = x.y; p[2] = x.z; p[3] = x.w; }
}

// Values of one row into the cache at `at`; `x` is this lane's part, element c + 4 * LANES * u + i in x[u] component i.
template <int DTYPE, int LANES, int U>
__device__ __forceinline__ void put_row(const float4 (&x)[U], void* cache, int64_t at, float* scale, int lane, int d, bool there, unsigned mask) {
    typedef typename Stored<DTYPE>::type S;
    S* row = static_cast<S*>(cache) + at;
    float inv = 1.0f;
    if constexpr (DTYPE == TE_KV_E4M3) {
        float amax = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float v[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) amax = fmaxf(amax, is_finite(v[i]) ? fabsf(v[i]) : 0.0f);
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(mask, amax, o));
        const int e = scale_exponent(amax);
        inv = power_of_two(-e);
        if (there && lane == 0) *scale = power_of_two(e);
    }
    if (!there) return;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int c = 4 * (lane + LANES * u);
        if (c >= d) continue;
        if constexpr (DTYPE == TE_KV_F32) {
            *reinterpret_cast<float4*>(row + c) = x[u];
        } else if constexpr (DTYPE == TE_KV_BF16) {
            __nv_bfloat162 lo = __floats2bfloat162_rn(x[u].x, x[u].y), hi = __floats2bfloat162_rn(x[u].z, x[u].w);
            uint2 w;
            w.x = *reinterpret_cast<unsigned*>(&lo);
            w.y = *reinterpret_cast<unsigned*>(&hi);
            *reinterpret_cast<uint2*>(row + c) = w;
        } else {
            // multiplying by the power of two rounds nothing that survives in 8 bits; the conversion rounds to nearest even
            const float v[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
            unsigned w = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __nv_fp8_storage_t q = __nv_cvt_float_to_fp8(is_finite(v[i]) ? v[i] * inv : __uint_as_float(0x7fc00000u), __NV_SATFINITE, __NV_E4M3);
                w |= (unsigned)q << (8 * i);
            }
            *reinterpret_cast<unsigned*>(row + c) = w;
        }
    }
}

template <int DTYPE>
__device__ __forceinline__ float4 get4(const typename Stored<DTYPE>::type* p, float scale) {
    if constexpr (DTYPE == TE_KV_F32) {
        return *reinterpret_cast<const float4*>(p);
    } else if constexpr (DTYPE == TE_KV_BF16) {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
    } else {
        const unsigned w = *reinterpret_cast<const unsigned*>(p);
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)(w >> (8 * i)), __NV_E4M3))) * scale;
        return make_float4(v[0], v[1], v[2], v[3]);
    }
}

// One group of lanes moves one row of k and the same row of v.
template <int DTYPE, int LANES, int U, bool VEC, bool APPEND>
__global__ void __launch_bounds__(256) kv_move_kernel(const KvParams p) {
    griddep_wait();
    constexpr int GROUPS = 256 / LANES;
    const int lane = threadIdx.x % LANES;
    const int64_t r = (int64_t)blockIdx.x * GROUPS + threadIdx.x / LANES;
    const unsigned mask = LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1u) << (threadIdx.x % 32 / LANES * LANES);
    if (r >= p.rows) return;                          // the whole group leaves
    const int64_t bh = r / p.T;
    const int t = (int)(r - bh * p.T);
    const int64_t b = bh / p.H;
    const int h = (int)(bh - b * p.H);
    float* k = p.k ? p.k + b * p.ks[0] + h * p.ks[1] + t * p.ks[2] : nullptr;
    float* v = p.v ? p.v + b * p.vs[0] + h * p.vs[1] + t * p.vs[2] : nullptr;
    const int64_t position = p.positions[b * p.ps[0] + t * p.ps[1]];
    const PageRow table = {p.page_table + b * p.table_stride, p.max_pages, p.pages};
    if constexpr (APPEND) {
        if (position < 0) return;                     // padding
        float4 x[U], y[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = 4 * (lane + LANES * u);
            x[u] = c < p.d ? load4<VEC>(k + c) : make_float4(0.f, 0.f, 0.f, 0.f);
            y[u] = c < p.d ? load4<VEC>(v + c) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        int64_t page = 0;
        uint32_t slot = 0;
        const bool there = kv_place(table, p.page_size, position, page, slot);
        if (!there) {
            if (lane == 0) atomicCAS(p.status, 0, STATUS_BAD_CACHE_PLACE);
            page = 0;
        }
        const int64_t s = DTYPE == TE_KV_E4M3 ? page * p.ss[0] + h * p.ss[1] + slot * p.ss[2] : 0;
        put_row<DTYPE, LANES, U>(x, p.kc, page * p.kcs[0] + h * p.kcs[1] + slot * p.kcs[2], p.k_scale + s, lane, p.d, there, mask);
        put_row<DTYPE, LANES, U>(y, p.vc, page * p.vcs[0] + h * p.vcs[1] + slot * p.vcs[2], p.v_scale + s, lane, p.d, there, mask);
    } else {
        typedef typename Stored<DTYPE>::type S;
        int64_t page = 0;
        uint32_t slot = 0;
        const bool there = kv_place(table, p.page_size, position, page, slot);
        if (!there && position >= 0 && lane == 0) atomicCAS(p.status, 0, STATUS_BAD_CACHE_PLACE);
        const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
        float4 x[U], y[U];
        float sk = 1.0f, sv = 1.0f;
        if (DTYPE == TE_KV_E4M3 && there) {
            const int64_t s = page * p.ss[0] + h * p.ss[1] + slot * p.ss[2];
            if (k) sk = p.k_scale[s];
            if (v) sv = p.v_scale[s];
        }
        const S* kr = static_cast<const S*>(p.kc) + page * p.kcs[0] + h * p.kcs[1] + slot * p.kcs[2];
        const S* vr = static_cast<const S*>(p.vc) + page * p.vcs[0] + h * p.vcs[1] + slot * p.vcs[2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = 4 * (lane + LANES * u);
            const bool in = there && c < p.d;
            x[u] = in && k ? get4<DTYPE>(kr + c, sk) : zero;
            y[u] = in && v ? get4<DTYPE>(vr + c, sv) : zero;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = 4 * (lane + LANES * u);
            if (c >= p.d) continue;
            if (k) store4<VEC>(k + c, x[u]);
            if (v) store4<VEC>(v + c, y[u]);
        }
    }
}

template <int DTYPE, bool APPEND>
cudaError_t launch_move(const KvParams& p, bool vec, cudaStream_t st) {
    const int lanes = p.d <= 32 ? 8 : p.d <= 64 ? 16 : 32;
    const int64_t groups = 256 / lanes;
    const dim3 grid((unsigned)((p.rows + groups - 1) / groups)), block(256);
#define TE_MOVE(L, U) (vec ? launch_pdl(kv_move_kernel<DTYPE, L, U, true, APPEND>, grid, block, 0, st, p) \
                           : launch_pdl(kv_move_kernel<DTYPE, L, U, false, APPEND>, grid, block, 0, st, p))
    if (lanes == 8) return TE_MOVE(8, 1);
    if (lanes == 16) return TE_MOVE(16, 1);
    return p.d <= 128 ? TE_MOVE(32, 1) : TE_MOVE(32, 2);
#undef TE_MOVE
}

bool vector_view(const float* p, const int64_t s[3]) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ((s[0] | s[1] | s[2]) & 3) == 0;
}

int move(te_b200_ctx* ctx, const te_kv_desc* t, bool append, cudaStream_t st) {
    const char* who = append ? "kv_append" : "kv_read";
    const std::string name = who;
    if (!t || t->B < 0 || t->T < 0 || t->max_pages < 0) return fail(TE_ERR_BAD_ARGUMENT, name + ": bad extents");
    if (int bad = check_kv_cache(t->cache, who)) return bad;
    const te_kv_cache& c = t->cache;
    if (t->max_pages > 0 && c.page_size > INT32_MAX / t->max_pages) return fail(TE_ERR_BAD_ARGUMENT, name + ": the page table reaches beyond 2^31-1 positions");
    if (t->T > INT32_MAX || t->B > INT32_MAX) return fail(TE_ERR_BAD_ARGUMENT, name + ": extent exceeds 2^31-1");
    const bool empty = t->B == 0 || t->T == 0 || c.heads == 0;
    if (!empty) {
        if (!t->positions || (t->max_pages > 0 && !t->page_table)) return fail(TE_ERR_BAD_ARGUMENT, name + ": NULL pointer");
        if (append ? (!t->k || !t->v) : (!t->k && !t->v)) return fail(TE_ERR_BAD_ARGUMENT, name + ": NULL pointer");
        if (t->page_table_stride < 0 || t->position_strides[0] < 0 || t->position_strides[1] < 0) return fail(TE_ERR_BAD_ARGUMENT, name + ": negative stride");
        const int64_t ext[3] = {t->B, c.heads, t->T};
        for (int i = 0; i < 3; ++i) {
            if (t->k_strides[i] < 0 || t->v_strides[i] < 0) return fail(TE_ERR_BAD_ARGUMENT, name + ": negative stride");
            if (!append && ext[i] > 1 && ((t->k && t->k_strides[i] < c.d) || (t->v && t->v_strides[i] < c.d)))
                return fail(TE_ERR_UNSUPPORTED_LAYOUT, name + ": rows of the output overlap");
        }
        // B, T < 2^31 each: bound their product before the heads come in
        if ((double)t->B * (double)t->T * (double)c.heads / 8.0 > 2147483647.0) return fail(TE_ERR_BAD_ARGUMENT, name + ": too many rows");
    }
    if (int bad = check_ctx(ctx)) return bad;
    if (empty) return TE_OK;
    KvParams p;
    p.k = t->k; p.v = t->v; p.kc = c.k; p.vc = c.v; p.k_scale = c.k_scale; p.v_scale = c.v_scale;
    p.page_table = t->page_table; p.positions = t->positions;
    for (int i = 0; i < 3; ++i) {
        p.ks[i] = t->k_strides[i]; p.vs[i] = t->v_strides[i];
        p.kcs[i] = c.k_strides[i]; p.vcs[i] = c.v_strides[i]; p.ss[i] = c.scale_strides[i];
    }
    p.ps[0] = t->position_strides[0]; p.ps[1] = t->position_strides[1];
    p.table_stride = t->page_table_stride; p.max_pages = t->max_pages; p.pages = c.pages;
    p.rows = t->B * c.heads * t->T;
    p.page_size = make_fast_divisor((uint32_t)c.page_size);
    p.T = (int)t->T; p.H = (int)c.heads; p.d = (int)c.d;
    p.status = ctx->d_status;
    const bool vec = (!t->k || vector_view(t->k, t->k_strides)) && (!t->v || vector_view(t->v, t->v_strides));
    cudaError_t e;
    if (c.dtype == TE_KV_F32) e = append ? launch_move<TE_KV_F32, true>(p, vec, st) : launch_move<TE_KV_F32, false>(p, vec, st);
    else if (c.dtype == TE_KV_BF16) e = append ? launch_move<TE_KV_BF16, true>(p, vec, st) : launch_move<TE_KV_BF16, false>(p, vec, st);
    else e = append ? launch_move<TE_KV_E4M3, true>(p, vec, st) : launch_move<TE_KV_E4M3, false>(p, vec, st);
    if (e != cudaSuccess) return cuda_fail(e, "kv_move_kernel launch");
    ctx->launches += 1;
    return TE_OK;
}

}  // namespace

int check_kv_cache(const te_kv_cache& c, const char* who) {
    const std::string name = who;
    if (c.dtype < TE_KV_F32 || c.dtype > TE_KV_E4M3) return fail(TE_ERR_BAD_ARGUMENT, name + ": cache dtype must be a TE_KV_* value");
    if (c.pages < 0 || c.heads < 0) return fail(TE_ERR_BAD_ARGUMENT, name + ": bad cache extents");
    if (c.heads > 65535) return fail(TE_ERR_BAD_ARGUMENT, name + ": more than 65535 cache heads");
    if (c.page_size < 1 || c.page_size > INT32_MAX) return fail(TE_ERR_BAD_ARGUMENT, name + ": page_size must be between 1 and 2^31-1");
    if (c.d < 16 || c.d > 256 || c.d % 16) return fail(TE_ERR_BAD_ARGUMENT, name + ": d must be a multiple of 16 between 16 and 256");
    if (c.pages > 0 && c.heads > 0) {
        if (!c.k || !c.v) return fail(TE_ERR_BAD_ARGUMENT, name + ": NULL cache pointer");
        if (c.dtype == TE_KV_E4M3 && (!c.k_scale || !c.v_scale)) return fail(TE_ERR_BAD_ARGUMENT, name + ": an 8-bit cache needs its scales");
    }
    const int64_t unit = c.dtype == TE_KV_F32 ? 4 : c.dtype == TE_KV_BF16 ? 8 : 16;      // elements in 16 bytes
    if (((reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v)) & 15) != 0)
        return fail(TE_ERR_UNSUPPORTED_LAYOUT, name + ": cache pointers must be 16-byte aligned");
    for (int i = 0; i < 3; ++i) {
        if (c.k_strides[i] < 0 || c.v_strides[i] < 0 || c.scale_strides[i] < 0) return fail(TE_ERR_BAD_ARGUMENT, name + ": negative cache stride");
        if (c.k_strides[i] % unit || c.v_strides[i] % unit) return fail(TE_ERR_UNSUPPORTED_LAYOUT, name + ": cache strides must be multiples of 16 bytes");
    }
    return TE_OK;
}

}  // namespace te

extern "C" {

int te_b200_kv_append(te_b200_ctx* ctx, const te_kv_desc* d, te_stream_t stream) {
    return te::move(ctx, d, true, static_cast<cudaStream_t>(stream));
}

int te_b200_kv_read(te_b200_ctx* ctx, const te_kv_desc* d, te_stream_t stream) {
    return te::move(ctx, d, false, static_cast<cudaStream_t>(stream));
}

}  // extern "C"

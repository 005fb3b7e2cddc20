// The paged key-value cache: tokens written into it (rounded to the cache's type, 8-bit rows with a power-of-two scale of
// their own) and read back as FP32.  Both directions are streaming kernels bound by HBM: 4 B of FP32 and 4, 2 or 1 B of
// cache per element (and 4 B of scale per 8-bit row).
//
// A row is the d elements of one (token, head) of k or of v.  A group of LANES lanes holds it, four elements a lane (eight
// for d > 128), so that FP32 moves in float4s, the largest magnitude of a row is one reduction within the group, and a
// row's bytes leave in one coalesced store.  A group moves ROWS consecutive tokens of one head (of k and of v) at once: they lie
// side by side in the cache's usual order [pages, heads, page_size, d], and their positions, page numbers and data are
// three loads one after the other that ROWS tokens wait for together.  Each lane works out the place of one of these
// tokens and the others take it from there.
//
// Measured (share of the 6.54 TB/s of a copy): FP32 [64,6,256,64] 18.0 us, 85 %; padded prompts [8,8,2001,128] into bf16 15.2 us,
// 79 % of what is not padding; [4,8,4093,128] into e4m3 and back 46 us, 79 %; 64 tokens of 8 heads 1.7 us, a launch's latency.
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
    FastDivisor page_size, blocks, heads;      // blocks: of ROWS tokens in T
    int tasks;                                 // B * H * blocks, the last fastest
    int T, d;
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

// Values of one row into the cache at `row`; `x` is this lane's part, element 4 * (lane + LANES * u) + i in x[u] component i.
template <int DTYPE, int LANES, int U>
__device__ __forceinline__ void put_row(const float4 (&x)[U], typename Stored<DTYPE>::type* row, float* scale, bool write_scale, int lane, int d, bool there, unsigned mask) {
    float inv = 1.0f;
    bool finite = true;
    if constexpr (DTYPE == TE_KV_E4M3) {
        unsigned top = 0u;             // magnitudes compare like their bits; those of what is not finite come last
#pragma unroll
        for (int u = 0; u < U; ++u)
            top = max(max(top, max(__float_as_uint(x[u].x) & 0x7fffffffu, __float_as_uint(x[u].y) & 0x7fffffffu)),
                      max(__float_as_uint(x[u].z) & 0x7fffffffu, __float_as_uint(x[u].w) & 0x7fffffffu));
        top = __reduce_max_sync(mask, top);
        finite = top < 0x7f800000u;
        if (!finite) {                 // (the whole group together)
            top = 0u;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float v[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) top = max(top, is_finite(v[i]) ? __float_as_uint(v[i]) & 0x7fffffffu : 0u);
            }
            top = __reduce_max_sync(mask, top);
        }
        const int e = scale_exponent(__uint_as_float(top));
        inv = power_of_two(-e);
        if (write_scale) *scale = power_of_two(e);
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
            float4 y = x[u];
            if (!finite) {
                const float nan = __uint_as_float(0x7fc00000u);
                y.x = is_finite(y.x) ? y.x : nan; y.y = is_finite(y.y) ? y.y : nan; y.z = is_finite(y.z) ? y.z : nan; y.w = is_finite(y.w) ? y.w : nan;
            }
            const unsigned lo = __nv_cvt_float2_to_fp8x2(make_float2(y.x * inv, y.y * inv), __NV_SATFINITE, __NV_E4M3);
            const unsigned hi = __nv_cvt_float2_to_fp8x2(make_float2(y.z * inv, y.w * inv), __NV_SATFINITE, __NV_E4M3);
            *reinterpret_cast<unsigned*>(row + c) = lo | hi << 16;
        }
    }
}

// Four elements as they are stored, and as FP32.
template <int DTYPE> struct Raw { typedef float4 type; };
template <> struct Raw<TE_KV_BF16> { typedef uint2 type; };
template <> struct Raw<TE_KV_E4M3> { typedef unsigned type; };
template <int DTYPE>
__device__ __forceinline__ float4 values_of(const typename Raw<DTYPE>::type& w, float scale) {
    if constexpr (DTYPE == TE_KV_F32) {
        return w;
    } else if constexpr (DTYPE == TE_KV_BF16) {
        return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
    } else {
        const float2 lo = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3)));
        const float2 hi = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3)));
        return make_float4(lo.x * scale, lo.y * scale, hi.x * scale, hi.y * scale);
    }
}

template <int DTYPE, int LANES, int U, int ROWS, bool VEC, bool APPEND>
__global__ void __launch_bounds__(256) kv_move_kernel(const KvParams p) {
    griddep_wait();
    typedef typename Stored<DTYPE>::type S;
    typedef typename Raw<DTYPE>::type W;
    constexpr int GROUPS = 256 / LANES;
    static_assert(ROWS <= LANES, "a lane per token");
    const int lane = threadIdx.x % LANES;
    const unsigned task = blockIdx.x * GROUPS + threadIdx.x / LANES;
    const int first_lane = threadIdx.x % 32 / LANES * LANES;
    const unsigned mask = LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1u) << first_lane;
    if (task >= (unsigned)p.tasks) return;            // the whole group leaves
    const unsigned bh = fast_quotient(task, p.blocks);
    const int t0 = (int)(task - bh * p.blocks.divisor) * ROWS;
    const unsigned b = fast_quotient(bh, p.heads);
    const int h = (int)(bh - b * p.heads.divisor);
    const int64_t* positions = p.positions + b * p.ps[0];
    const int own = lane % ROWS;                       // the token whose place this lane works out
    const int64_t position = t0 + own < p.T ? positions[(t0 + own) * p.ps[1]] : -1;
    const unsigned wanted = __ballot_sync(mask, position >= 0) >> first_lane;        // not padding: bit i for token i
    if (APPEND && (wanted & ((1u << ROWS) - 1u)) == 0u) return;
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    float4 x[APPEND ? ROWS : 1][U], y[APPEND ? ROWS : 1][U];
    float* k = p.k + b * p.ks[0] + h * p.ks[1] + t0 * p.ks[2] + 4 * lane;
    float* v = p.v + b * p.vs[0] + h * p.vs[1] + t0 * p.vs[2] + 4 * lane;
    if constexpr (APPEND) {
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool in = (wanted >> i & 1u) && 4 * (lane + LANES * u) < p.d;       // (nothing is read of padding)
                x[i][u] = in ? load4<VEC>(k + i * p.ks[2] + 4 * LANES * u) : zero;
                y[i][u] = in ? load4<VEC>(v + i * p.vs[2] + 4 * LANES * u) : zero;
            }
    }
    const PageRow table = {p.page_table + b * p.table_stride, p.max_pages, p.pages};
    int64_t page = 0;
    uint32_t slot = 0;
    const bool found = kv_place(table, p.page_size, position, page, slot);
    if (!found && position >= 0 && lane < ROWS) atomicCAS(p.status, 0, STATUS_BAD_CACHE_PLACE);
    const unsigned there = __ballot_sync(mask, found) >> first_lane;
    const unsigned at = found ? (unsigned)page : 0u;   // (pages of a cache are below 2^31)
    if (!found) slot = 0u;
    const long long ka = at * p.kcs[0] + slot * p.kcs[2], va = at * p.vcs[0] + slot * p.vcs[2];
    S* kc = static_cast<S*>(p.kc) + h * p.kcs[1];
    S* vc = static_cast<S*>(p.vc) + h * p.vcs[1];
    const int64_t sa = DTYPE == TE_KV_E4M3 ? at * p.ss[0] + h * p.ss[1] + slot * p.ss[2] : 0;
    if constexpr (APPEND) {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const bool to = there >> i & 1u;
            const long long kr = __shfl_sync(mask, ka, first_lane + i), vr = __shfl_sync(mask, va, first_lane + i);
            put_row<DTYPE, LANES, U>(x[i], kc + kr, p.k_scale + sa, to && lane == i, lane, p.d, to, mask);
            put_row<DTYPE, LANES, U>(y[i], vc + vr, p.v_scale + sa, to && lane == i, lane, p.d, to, mask);
        }
    } else {
        W kw[ROWS][U] = {}, vw[ROWS][U] = {};
        float ks = 1.0f, vs = 1.0f;
        if (DTYPE == TE_KV_E4M3 && found) {
            if (p.k) ks = p.k_scale[sa];
            if (p.v) vs = p.v_scale[sa];
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const long long kr = __shfl_sync(mask, ka, first_lane + i), vr = __shfl_sync(mask, va, first_lane + i);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = 4 * (lane + LANES * u);
                const bool in = (there >> i & 1u) && c < p.d;
                if (in && p.k) kw[i][u] = *reinterpret_cast<const W*>(kc + kr + c);
                if (in && p.v) vw[i][u] = *reinterpret_cast<const W*>(vc + vr + c);
            }
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const float sk = DTYPE == TE_KV_E4M3 ? __shfl_sync(mask, ks, first_lane + i) : 1.0f;
            const float sv = DTYPE == TE_KV_E4M3 ? __shfl_sync(mask, vs, first_lane + i) : 1.0f;
            if (t0 + i >= p.T) continue;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (4 * (lane + LANES * u) >= p.d) continue;
                if (p.k) store4<VEC>(k + i * p.ks[2] + 4 * LANES * u, values_of<DTYPE>(kw[i][u], sk));
                if (p.v) store4<VEC>(v + i * p.vs[2] + 4 * LANES * u, values_of<DTYPE>(vw[i][u], sv));
            }
        }
    }
}

// Tokens a group moves at once: one where there are few per sequence; else two rows of FP32 in and out (17.5 us for
// [64,6,256,64], 17.9 with four), or up to four (written; padded bf16 prompts 15.2 us, 16.2 with two) or eight (read) of the
// narrower types.
constexpr int MOST_F32 = 2, MOST_APPENDED = 4, MOST_READ = 8;
int rows_at_once(int dtype, int T, int d, bool append) {
    if (T < 4) return 1;
    return dtype == TE_KV_F32 || d > 128 ? MOST_F32 : append ? MOST_APPENDED : MOST_READ;
}

template <int DTYPE, bool APPEND>
cudaError_t launch_move(const KvParams& p, bool vec, cudaStream_t st) {
    constexpr int MANY = DTYPE == TE_KV_F32 ? MOST_F32 : APPEND ? MOST_APPENDED : MOST_READ;
    const int lanes = p.d <= 32 ? 8 : p.d <= 64 ? 16 : 32, rows = rows_at_once(DTYPE, p.T, p.d, APPEND);
    const int groups = 256 / lanes;
    const dim3 grid((unsigned)(((unsigned)p.tasks + groups - 1) / groups)), block(256);
#define TE_MOVE(L, U, N) (vec ? launch_pdl(kv_move_kernel<DTYPE, L, U, N, true, APPEND>, grid, block, 0, st, p) \
                              : launch_pdl(kv_move_kernel<DTYPE, L, U, N, false, APPEND>, grid, block, 0, st, p))
    if (lanes == 8) return rows == 1 ? TE_MOVE(8, 1, 1) : TE_MOVE(8, 1, MANY);
    if (lanes == 16) return rows == 1 ? TE_MOVE(16, 1, 1) : TE_MOVE(16, 1, MANY);
    if (p.d <= 128) return rows == 1 ? TE_MOVE(32, 1, 1) : TE_MOVE(32, 1, MANY);
    return rows == 1 ? TE_MOVE(32, 2, 1) : TE_MOVE(32, 2, MOST_F32);
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
        if ((double)t->B * (double)t->T * (double)c.heads > 2147483000.0) return fail(TE_ERR_BAD_ARGUMENT, name + ": too many rows");
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
    p.page_size = make_fast_divisor((uint32_t)c.page_size);
    p.T = (int)t->T; p.d = (int)c.d;
    const int rows = rows_at_once(c.dtype, p.T, p.d, append);
    p.blocks = make_fast_divisor((uint32_t)((p.T + rows - 1) / rows));
    p.heads = make_fast_divisor((uint32_t)c.heads);
    p.tasks = (int)(t->B * c.heads * p.blocks.divisor);
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
    if (c.pages > INT32_MAX) return fail(TE_ERR_BAD_ARGUMENT, name + ": more than 2^31-1 pages");
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

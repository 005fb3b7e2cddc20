// Rotary positions: pairs of a head's elements turned by angle position * inv_freq[pair], forward and (turned back) backward.
//
//     (y0, y1) = scale * (x0 cos a - x1 sin a, x0 sin a + x1 cos a)
//
// Bound by HBM: 4 B read and 4 B written per element.  The angle is the same for every head of a token, so a thread keeps
// the cosines and sines of its pairs in registers and walks the heads with them; nothing goes through shared memory and no
// thread waits for another.  Angles: position * inv_freq is formed and reduced to a fraction of a turn in FP64 (an FP32
// product is off by 2^-24 of the whole angle, 0.06 rad at position 10^6); the fraction, below one half, goes to
// sincospif in FP32.
//
// Measured (share of the 6.54 TB/s of a copy): q and k views [64,12,256,64] inside a projections' buffer 19.5 us, 79 %;
// backward, interleaved, half of the head, [1,32,8191,128] 49 us, 83 %; eight tokens of 40 heads 2.3 us, a launch's latency.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "pdl.cuh"
#include "te_internal.h"

namespace te {

namespace {

struct RotaryParams {
    const float* x;
    float* y;
    const long long* positions;
    const double* inv_freq;
    long long xs[3], ys[3], ps[2];
    long long total;             // threads with work: tokens * head_lanes * items
    int T, H, rot, d;
    int head_lanes;              // threads that share the heads of a (token, item)
    int rot_items, items;        // of a head: groups of W pairs, then of 2 W copied elements
    float scale, sign;
};

// A thread takes two vectors of W elements of every head of a token: W pairs, or 2 W elements behind the rotated part (where they
// are left as they are).  W = 4 moves float4s and needs rot in multiples of 8, d of 4, and aligned views.
template <int W> struct Vector { float x[W]; };
template <int W>
__device__ __forceinline__ void load(Vector<W>& v, const float* p) {
    if constexpr (W == 4) {
        const float4 t = __ldcs(reinterpret_cast<const float4*>(p));
        v.x[0] = t.x; v.x[1] = t.y; v.x[2] = t.z; v.x[3] = t.w;
    } else {
        v.x[0] = *p;
    }
}
template <int W>
__device__ __forceinline__ void store(float* p, const Vector<W>& v) {
    if constexpr (W == 4) *reinterpret_cast<float4*>(p) = make_float4(v.x[0], v.x[1], v.x[2], v.x[3]);
    else *p = v.x[0];
}

template <int W, bool INTERLEAVED>
__global__ void __launch_bounds__(256, 4) rotary_kernel(const RotaryParams p) {
    griddep_wait();
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= p.total) return;
    const unsigned rest = (unsigned)(i / p.items);          // (token, head lane): below 2^31
    const int item = (int)(i - (long long)rest * p.items);
    const unsigned token = rest / (unsigned)p.head_lanes;
    const int lane = (int)(rest - token * p.head_lanes);
    const unsigned b = token / (unsigned)p.T;
    const int t = (int)(token - b * p.T);
    const bool turned = item < p.rot_items;
    // Element offsets of the thread's two vectors, half the rotated (or the copied) part apart, so that a warp's accesses are
    // contiguous in either layout; and the pairs their elements belong to: W from j0, or (interleaved) W / 2 from j0 and from j1.
    int o0 = item * W, o1 = o0 + p.rot / 2;
    const int j0 = INTERLEAVED && W == 4 ? o0 / 2 : o0, j1 = INTERLEAVED && W == 4 ? o1 / 2 : 0;
    if (INTERLEAVED && W == 1) { o0 = 2 * item; o1 = o0 + 1; }
    if (!turned) {
        const int vectors = (p.d - p.rot) / W, half = (vectors + 1) / 2, k = item - p.rot_items;
        o0 = p.rot + k * W;
        o1 = k + half < vectors ? o0 + half * W : o0;        // (the last vector may be alone: moved twice)
    }
    const float* x = p.x + b * p.xs[0] + t * p.xs[2];
    float* y = p.y + b * p.ys[0] + t * p.ys[2];
    // several heads at a time; the first are under way while the angles are computed
    constexpr int N = 4;
    const int step = p.head_lanes;
    Vector<W> u[N], v[N];
    auto fetch = [&](int h) {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (h + k * step < p.H) {
                const float* xh = x + (h + k * step) * p.xs[1];
                load(u[k], xh + o0);
                load(v[k], xh + o1);
            }
    };
    fetch(lane);
    float c[W], s[W];
    if (turned) {
        const double position = (double)p.positions[b * p.ps[0] + t * p.ps[1]];
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const int j = INTERLEAVED && W == 4 && w >= 2 ? j1 + w - 2 : j0 + w;
            const double turns = position * p.inv_freq[j] * 0.15915494309189535;      // 1 / (2 pi)
            const float part = (float)(turns - rint(turns));
            sincospif(2.0f * part, &s[w], &c[w]);
            c[w] *= p.scale;
            s[w] *= p.scale * p.sign;
        }
    }
    for (int h = lane; h < p.H; h += N * step) {
        if (h != lane) fetch(h);
        if (turned) {
#pragma unroll
            for (int k = 0; k < N; ++k) {
                if constexpr (INTERLEAVED && W == 4) {
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const float a0 = u[k].x[2 * w], a1 = u[k].x[2 * w + 1], e0 = v[k].x[2 * w], e1 = v[k].x[2 * w + 1];
                        u[k].x[2 * w] = a0 * c[w] - a1 * s[w];
                        u[k].x[2 * w + 1] = a0 * s[w] + a1 * c[w];
                        v[k].x[2 * w] = e0 * c[w + 2] - e1 * s[w + 2];
                        v[k].x[2 * w + 1] = e0 * s[w + 2] + e1 * c[w + 2];
                    }
                } else {
#pragma unroll
                    for (int w = 0; w < W; ++w) {
                        const float a0 = u[k].x[w], e0 = v[k].x[w];
                        u[k].x[w] = a0 * c[w] - e0 * s[w];
                        v[k].x[w] = a0 * s[w] + e0 * c[w];
                    }
                }
            }
        }
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (h + k * step < p.H) {
                float* yh = y + (h + k * step) * p.ys[1];
                store(yh + o0, u[k]);
                store(yh + o1, v[k]);
            }
    }
}

bool vector_view(const float* p, const int64_t s[3]) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ((s[0] | s[1] | s[2]) & 3) == 0;
}

}  // namespace

}  // namespace te

using namespace te;

extern "C" {

int te_b200_rotary_inv_freq(int64_t rot, double base, int scaling, double factor, int64_t trained_length, double slow_turns,
                            double fast_turns, double* out) {
    if (rot < 0 || (rot & 1)) return fail(TE_ERR_BAD_ARGUMENT, "rotary: the rotated width must be even and not negative");
    if (!(base > 0.0)) return fail(TE_ERR_BAD_ARGUMENT, "rotary: base must be positive");
    if (scaling < TE_ROTARY_PLAIN || scaling > TE_ROTARY_PARTS) return fail(TE_ERR_BAD_ARGUMENT, "rotary: scaling must be a TE_ROTARY_* value");
    if (scaling != TE_ROTARY_PLAIN && !(factor > 0.0)) return fail(TE_ERR_BAD_ARGUMENT, "rotary: factor must be positive");
    if (scaling == TE_ROTARY_BASE && rot <= 2) return fail(TE_ERR_BAD_ARGUMENT, "rotary: TE_ROTARY_BASE needs more than one pair");
    if (scaling == TE_ROTARY_PARTS && (trained_length < 1 || !(fast_turns > slow_turns)))
        return fail(TE_ERR_BAD_ARGUMENT, "rotary: TE_ROTARY_PARTS needs trained_length >= 1 and fast_turns > slow_turns");
    if (rot > 0 && !out) return fail(TE_ERR_BAD_ARGUMENT, "rotary: NULL pointer");
    if (scaling == TE_ROTARY_BASE) base *= pow(factor, (double)rot / (double)(rot - 2));
    for (int64_t j = 0; j < rot / 2; ++j) {
        double f = pow(base, -2.0 * (double)j / (double)rot);
        if (scaling == TE_ROTARY_LINEAR) {
            f /= factor;
        } else if (scaling == TE_ROTARY_PARTS) {
            const double turns = (double)trained_length * f / 6.283185307179586;
            double keep = (turns - slow_turns) / (fast_turns - slow_turns);
            keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
            f *= keep + (1.0 - keep) / factor;
        }
        out[j] = f;
    }
    return TE_OK;
}

int te_b200_rotary(te_b200_ctx* ctx, const te_rotary_desc* t, te_stream_t stream) {
    if (!t || t->B < 0 || t->H < 0 || t->T < 0 || t->d < 0) return fail(TE_ERR_BAD_ARGUMENT, "rotary: bad extents");
    if (t->rot < 0 || (t->rot & 1) || t->rot > t->d) return fail(TE_ERR_BAD_ARGUMENT, "rotary: the rotated width must be even and at most d");
    if (t->d > 1024) return fail(TE_ERR_BAD_ARGUMENT, "rotary: heads longer than 1024 elements are not supported");
    if (t->H > INT32_MAX || t->T > INT32_MAX || (t->T > 0 && t->B > INT32_MAX / t->T)) return fail(TE_ERR_BAD_ARGUMENT, "rotary: extent exceeds 2^31-1");
    if (t->B > 0 && t->H > 0 && t->T > 0 && t->d > 0) {
        if (!t->x || !t->y || (t->rot > 0 && (!t->positions || !t->inv_freq))) return fail(TE_ERR_BAD_ARGUMENT, "rotary: NULL pointer");
        const int64_t ext[3] = {t->B, t->H, t->T};
        for (int i = 0; i < 3; ++i) {
            if (t->x_strides[i] < 0 || t->y_strides[i] < 0) return fail(TE_ERR_BAD_ARGUMENT, "rotary: negative stride");
            if (ext[i] > 1 && t->y_strides[i] < t->d) return fail(TE_ERR_UNSUPPORTED_LAYOUT, "rotary: heads of the output overlap");
            if (t->x == t->y && ext[i] > 1 && t->x_strides[i] != t->y_strides[i])
                return fail(TE_ERR_UNSUPPORTED_LAYOUT, "rotary: in place needs equal strides of input and output");
        }
        if (t->position_strides[0] < 0 || t->position_strides[1] < 0) return fail(TE_ERR_BAD_ARGUMENT, "rotary: negative stride");
    }
    if (int bad = check_ctx(ctx)) return bad;
    if (t->B == 0 || t->H == 0 || t->T == 0 || t->d == 0) return TE_OK;
    RotaryParams p;
    p.x = t->x; p.y = t->y;
    p.positions = reinterpret_cast<const long long*>(t->positions);
    p.inv_freq = t->inv_freq;
    for (int i = 0; i < 3; ++i) { p.xs[i] = t->x_strides[i]; p.ys[i] = t->y_strides[i]; }
    p.ps[0] = t->position_strides[0]; p.ps[1] = t->position_strides[1];
    p.T = (int)t->T; p.H = (int)t->H; p.rot = (int)t->rot; p.d = (int)t->d;
    p.scale = t->scale;
    p.sign = t->inverse ? -1.0f : 1.0f;
    const bool vec = vector_view(t->x, t->x_strides) && vector_view(t->y, t->y_strides) && p.rot % 8 == 0 && p.d % 4 == 0;
    const int w = vec ? 4 : 1;
    p.rot_items = p.rot / (2 * w);
    p.items = p.rot_items + (t->x == t->y ? 0 : (p.d - p.rot + 2 * w - 1) / (2 * w));
    if (p.items == 0) return TE_OK;                  // in place with nothing to turn
    // One thread per (token, item) where that fills the GPU (four blocks of 256 threads per SM); otherwise its heads are shared
    // among several.
    const long long tokens = t->B * t->T, base = tokens * p.items, fill = (long long)ctx->sm_count * 1024;
    long long lanes = fill / base;
    lanes = lanes < 1 ? 1 : lanes > p.H ? p.H : lanes;
    p.head_lanes = (int)lanes;
    p.total = base * p.head_lanes;
    const long long blocks = (p.total + 255) / 256;
    if (blocks > INT32_MAX) return fail(TE_ERR_BAD_ARGUMENT, "rotary: too many elements");
    const dim3 grid((unsigned)blocks), block(256);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (vec) e = t->interleaved ? launch_pdl(rotary_kernel<4, true>, grid, block, 0, st, p) : launch_pdl(rotary_kernel<4, false>, grid, block, 0, st, p);
    else e = t->interleaved ? launch_pdl(rotary_kernel<1, true>, grid, block, 0, st, p) : launch_pdl(rotary_kernel<1, false>, grid, block, 0, st, p);
    if (e != cudaSuccess) return cuda_fail(e, "rotary_kernel launch");
    ctx->launches += 1;
    return TE_OK;
}

}  // extern "C"

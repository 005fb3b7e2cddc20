// Attention of one new token per row over a paged key-value cache.
//
//     o = sum_t p_t v_t / sum_t p_t,   p_t = exp(scale * q . k_t - m),   m the running maximum
//
// Bound by reading the cache once: 2 d values of 4, 2 or 1 byte per cached token and key head.  What follows from that:
//
// * Query heads that share a key head are computed together (up to 8, a head tile), so that a value is read once for all.
// * A fixed number of thread blocks, all resident, share the tiles of all rows evenly (paged_plan.h), so that one long
//   sequence, many short ones and any mixture keep every SM reading.  A block that holds only part of a (row, head tile)
//   leaves its sums in the workspace; paged_join_kernel adds the parts in their order.
// * Every warp copies its own tokens into a ring of its own in shared memory, 16 bytes a lane with cp.async, one or two stages
//   ahead of the one it computes on and on into its next segments, and waits for nobody else until a segment ends.
//
// 2- and 1-byte caches use the tensor cores through mma.sync m16n8k16 (8 query rows do not fill the 128-row tiles of
// tcgen05, and the tensor pipe is 20 to 35 % busy): a stored value is exactly a bf16 resp. half, and an FP32 query or
// weight is, to 2^-24 of its row's largest, the sum of three bf16 resp. two half terms, so that products and sums are
// those of FP32 (relative error against 64 bits 2e-7 to 4e-7).  The terms of a head occupy rows g and g + 8 of one tile,
// both in the same thread.  Which element of a head an index of the contraction stands for is free as long as both
// operands agree, and chosen so that a lane's operand is 16 bytes of a row as it lies in the cache.  An FP32 cache uses
// FP32 FMAs (two per instruction).
//
// Measured (device time, share of the 6.54 TB/s of a copy): 32 rows of 164 to 16384 tokens, 32 query and 8 key heads of 128,
// bf16: 86 us, 94 %; two rows of up to 131072 tokens, 64/8 heads, e4m3: 74 us, 82 % (bound by instruction issue: every
// stored value is converted); 16 rows, 20 heads of 80, pages of 13, window 4096, bf16: 40 us, 68 % (places looked up token by
// token); 64 FP32 rows of up to 1024 tokens, 6 heads of 64: 15 us, 50 %, and one of 200 tokens: 6 us (a chain of loads:
// lengths, page table, keys, parts).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "paged_plan.h"
#include "pdl.cuh"
#include "te_internal.h"

namespace te {

namespace {

constexpr int WARPS = 4;
constexpr int THREADS = 32 * WARPS;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// Thread blocks per SM, as registers and rings allow.  bf16 rows of up to 256 bytes and FP32 tiles of one or two heads do with 168
// registers a thread, so three blocks with two stages each (window of 4096 bf16 tokens: 48 us against 52 with two blocks
// of three stages).  e4m3 spills at 168 (two 131072-token rows: 75 us against 74), wide FP32 tiles too: two blocks.  Two rings of
// the longest rows do not fit: one block.
constexpr int blocks_per_sm(int dtype, int d, int heads) {
    return dtype == TE_KV_E4M3 ? 2 : d > 128 ? 1 : dtype == TE_KV_BF16 || heads <= 2 ? 3 : 2;
}

struct AttnParams {
    const float* q;
    float* o;
    float* lse;
    const char* kc;
    const char* vc;
    const float* k_scale;
    const float* v_scale;
    const int64_t* page_table;
    const int64_t* lens;
    int64_t qs[2], os[2];
    int64_t kcs[3], vcs[3];       // bytes
    int64_t ss[3];                // elements
    int64_t table_stride, pages, window;
    FastDivisor page_size;
    int most;                     // positions the page table reaches
    int rows, q_heads, kv_heads, group, head_tiles, d;
    float scale;
    float* part_acc;              // [2 * workers][heads of a tile][d]
    float2* part_ml;              // [2 * workers][heads of a tile]: running maximum (base 2) and sum
    int4* joins;                  // [workers]: row, head tile, last worker, 1 -- of the segment that begins in this share and is split
    int* arrived;                 // [workers] counters, zero between launches: parts done of the segment that begins in a share; NULL
                                  // where paged_join_kernel adds the parts
    int* status;
};

struct Heads {
    int kv_head, head0, count;       // query heads head0 .. head0 + count - 1
};
template <int HT>
__device__ __forceinline__ Heads heads_of(const AttnParams& p, int head_tile) {
    Heads h;
    h.kv_head = p.head_tiles == 1 ? head_tile : head_tile / p.head_tiles;
    const int part = (head_tile - h.kv_head * p.head_tiles) * HT;
    h.head0 = h.kv_head * p.group + part;
    h.count = min(HT, p.group - part);
    return h;
}

// ---------------------------------------------------------------------------------------------------- small pieces
// c += a b, and c = a b; a holds the four words of the left operand.
template <bool HALF>
__device__ __forceinline__ void mma(float (&c)[4], const uint4& a, unsigned b0, unsigned b1) {
    if constexpr (HALF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
template <bool HALF>
__device__ __forceinline__ void mma_from_zero(float (&c)[4], const uint4& a, unsigned b0, unsigned b1) {
    if constexpr (HALF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(0.0f));
}
template <bool HALF>
__device__ __forceinline__ void mma_first_or_next(bool first, float (&c)[4], const uint4& a, unsigned b0, unsigned b1) {
    if (first) mma_from_zero<HALF>(c, a, b0, b1);
    else mma<HALF>(c, a, b0, b1);
}
__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&v);
}
__device__ __forceinline__ float bf16_lo(unsigned v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_hi(unsigned v) { return __uint_as_float(v & 0xffff0000u); }
__device__ __forceinline__ unsigned pack_half(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&v);
}
__device__ __forceinline__ float2 unpack_half(unsigned v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
// Four e4m3 values (low byte first) as four halves, exactly.
__device__ __forceinline__ uint2 halves_of_e4m3(unsigned four) {
    uint2 r;
    asm("{ .reg .b16 lo, hi; mov.b32 {lo, hi}, %2; cvt.rn.f16x2.e4m3x2 %0, lo; cvt.rn.f16x2.e4m3x2 %1, hi; }" : "=r"(r.x), "=r"(r.y) : "r"(four));
    return r;
}
__device__ __forceinline__ unsigned smem_address(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(unsigned to, const char* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// Zeros where !there (nothing is read then).
__device__ __forceinline__ void copy16_or_zero(unsigned to, const char* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4_or_zero(unsigned to, const float* from, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ unsigned long long pair(float x, float y) {
    unsigned long long v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
    return v;
}
__device__ __forceinline__ float2 unpair(unsigned long long v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ void fma2(unsigned long long& d, unsigned long long a, unsigned long long b) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(d) : "l"(a), "l"(b));
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// 2^x to 2^-22 of itself, denormal results flushed: they are weights next to one of 1.
__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// What is taken from a score before exp2_of: the maximum; one of -infinity means that nothing has been seen.
__device__ __forceinline__ float settled(float m) { return m == -INFINITY ? 0.0f : m; }

// A warp's ring: stages of TOKENS rows of keys and as many of values (and their scales), DP elements of ES bytes a row.
//
// PACKED: pages are multiples of 16 slots, rows of a page and head lie one behind the other, and d == DP.  Sixteen tokens
// are then one contiguous piece, and a stage's copies are immediate offsets from a few page addresses.  Otherwise every
// token's place is looked up by the lane of its number and handed round, and what a row lacks to DP elements is zero-filled.
//
// Rows are multiples of 128 bytes apart (of 64 for DP = 64 bytes), so lanes that read different rows would meet in the
// same banks.  16-byte pieces are therefore exchanged within a row by an exclusive-or with bits of the row's number:
// readers of keys take pieces 4c .. 4c + 3 of rows 2i and 2i + 1 at a time, readers of values pieces 2c, 2c + 1 of every
// other row of eight.
template <int DP, int ES, int TOKENS_, int STAGES_, bool SCALES, bool PACKED>
struct Ring {
    static constexpr int TOKENS = TOKENS_, STAGES = STAGES_;
    static constexpr int RB = DP * ES;                                 // bytes of a row
    static constexpr int CPR = RB / 16;                                // pieces of a row
    static constexpr int TPI = CPR >= 32 ? 1 : 32 / CPR;               // rows a warp copies at once
    static constexpr int PPR = CPR >= 32 ? CPR / 32 : 1;               // copies a lane makes of a row
    static constexpr int SIDE = TOKENS * RB;                           // bytes of the keys, and of the values, of a stage
    static constexpr int STAGE = 2 * SIDE + (SCALES ? 2 * TOKENS * 4 : 0);
    static constexpr int BYTES = STAGE * STAGES;
    static constexpr int STEP = WARPS * TOKENS;                        // from one of a warp's stages to its next
    static constexpr int BLOCK = TOKENS < 16 ? TOKENS : 16;            // tokens of one page lookup
    static constexpr int NB = PACKED ? TOKENS / BLOCK : 1;

    // Byte offset of piece j of row t.
    static __device__ __forceinline__ int key_at(int t, int j) {
        return RB == 64 ? ((t * 4 + j) ^ ((t >> 1 & 1) << 1) ^ ((t >> 2 & 1) << 2)) * 16 : t * RB + (j ^ ((t & 1) << 2)) * 16;
    }
    static __device__ __forceinline__ int value_at(int t, int j) {
        if constexpr (ES == 4) return t * RB + j * 16;                 // lanes read along a row
        return RB == 64 ? key_at(t, j) : t * RB + (j ^ ((t >> 1 & 3) << 1)) * 16;
    }

    unsigned base;              // shared-memory address of the ring
    int64_t entry[NB];          // of the page table, as read, for the stage to be issued next
    unsigned slot[NB];

    // Reads the page table for the tokens from t0 on; lane's own token (!PACKED), or the page of each block.
    __device__ __forceinline__ void look_up(const AttnParams& p, const int64_t* table, int t0, int n) {
        const int lane = threadIdx.x % 32;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int t = t0 + (PACKED ? b * BLOCK : lane % TOKENS);
            entry[b] = -1;
            slot[b] = 0;
            if (t < n) {                               // n is within the table
                const unsigned i = fast_quotient((unsigned)t, p.page_size);
                slot[b] = (unsigned)t - i * p.page_size.divisor;
                entry[b] = __ldg(table + i);
            }
        }
    }

    // Issues the copies of the tokens from t0 on, whose places look_up has read, into stage i.  Returns which of them may be
    // attended to: bit t for token t0 + t.
    __device__ __forceinline__ unsigned issue(const AttnParams& p, const RowRange& range, int kv_head, int t0, int i) {
        const int lane = threadIdx.x % 32;
        const unsigned to = base + i * STAGE;
        const int chunk = lane % (CPR < 32 ? CPR : 32), sub = CPR >= 32 ? 0 : lane / CPR;
        const char* kc = p.kc + kv_head * p.kcs[1];
        const char* vc = p.vc + kv_head * p.vcs[1];
        // tokens inside the range, then those on pages of the cache
        constexpr unsigned ALL = 0xffffffffu >> (32 - TOKENS);
        const int lo = range.first - t0, hi = range.n - t0;
        unsigned seen = ALL;
        if (lo > 0 || hi < TOKENS) {
            seen = hi <= 0 ? 0u : hi >= TOKENS ? ALL : (1u << hi) - 1u;
            if (lo > 0) seen = lo >= TOKENS ? 0u : seen & ~((1u << lo) - 1u);
        }
        unsigned good = 0u;
        if constexpr (PACKED) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
                if (entry[b] >= 0 && entry[b] < p.pages) good |= (BLOCK == 16 ? 0xffffu : 0xffu) << (b * BLOCK);
        } else {
            good = __ballot_sync(0xffffffffu, entry[0] >= 0 && entry[0] < p.pages);
        }
        if (seen & ~good) {
            if (lane == 0) atomicCAS(p.status, 0, STATUS_BAD_CACHE_PLACE);
            seen &= good;
        }
        if constexpr (PACKED) {
            const char *k[NB], *v[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const bool there = (good >> (b * BLOCK)) & 1u;
                k[b] = kc + (there ? (unsigned)entry[b] * p.kcs[0] + (unsigned long long)slot[b] * RB : 0) + lane * 16;
                v[b] = vc + (there ? (unsigned)entry[b] * p.vcs[0] + (unsigned long long)slot[b] * RB : 0) + lane * 16;
            }
            auto copy = [&](auto whole) {
#pragma unroll
                for (int i = 0; i < TOKENS / TPI * PPR; ++i) {
                    const int u = i % PPR, t = i / PPR * TPI + sub;                                     // (t: lane's token)
                    constexpr int PER = BLOCK / TPI * PPR;
                    const unsigned kd = to + key_at(t, chunk + 32 * u), vd = to + SIDE + value_at(t, chunk + 32 * u);
                    const char* from_k = k[i / PER] + i % PER * 512;
                    const char* from_v = v[i / PER] + i % PER * 512;
                    if constexpr (decltype(whole)::value) {
                        copy16(kd, from_k);
                        copy16(vd, from_v);
                    } else {
                        copy16_or_zero(kd, from_k, seen >> t & 1u);
                        copy16_or_zero(vd, from_v, seen >> t & 1u);
                    }
                }
            };
            if (seen == ALL) copy(std::true_type());
            else copy(std::false_type());
        } else {
            const unsigned page = good >> lane & 1u ? (unsigned)entry[0] : 0u;
            const long long ko = page * p.kcs[0] + slot[0] * p.kcs[2], vo = page * p.vcs[0] + slot[0] * p.vcs[2];
            const bool same = p.kcs[0] == p.vcs[0] && p.kcs[2] == p.vcs[2];
            const int width = p.d * ES;
            auto copy = [&](auto same_places) {
#pragma unroll
                for (int c = 0; c < TOKENS / TPI; ++c) {
                    const int t = c * TPI + sub;
                    const long long k = __shfl_sync(0xffffffffu, ko, t);
                    const long long v = decltype(same_places)::value ? k : __shfl_sync(0xffffffffu, vo, t);
#pragma unroll
                    for (int u = 0; u < PPR; ++u) {
                        const int j = chunk + 32 * u;
                        const bool there = (seen >> t & 1u) && j * 16 < width;
                        const int byte = there ? j * 16 : 0;
                        copy16_or_zero(to + key_at(t, j), kc + k + byte, there);
                        copy16_or_zero(to + SIDE + value_at(t, j), vc + v + byte, there);
                    }
                }
            };
            if (same) copy(std::true_type());
            else copy(std::false_type());
        }
        if constexpr (SCALES) {          // lane t copies token t's
            int64_t at = 0;
            const bool mine = lane < TOKENS && (seen >> (lane % TOKENS) & 1u);
            if constexpr (PACKED) {
                const bool second = NB > 1 && lane >= BLOCK;
                at = (second ? (unsigned)entry[NB - 1] : (unsigned)entry[0]) * p.ss[0] + ((second ? slot[NB - 1] : slot[0]) + lane % BLOCK) * p.ss[2];
            } else {
                at = entry[0] * p.ss[0] + (int64_t)slot[0] * p.ss[2];
            }
            at = mine ? at + kv_head * p.ss[1] : 0;
            if (lane < TOKENS) {
                copy4_or_zero(to + 2 * SIDE + lane * 4, p.k_scale + at, mine);
                copy4_or_zero(to + 2 * SIDE + TOKENS * 4 + lane * 4, p.v_scale + at, mine);
            }
        }
        return seen;
    }
};

// ------------------------------------------------------------------------------------------- 2- and 1-byte caches
// One warp's share of a segment on the tensor cores, 16 or 32 tokens at a time.
//
// Lane (g, r) = (lane / 4, lane % 4).  Scores S = Q K^T: the lane's operand of K is 16 bytes of tokens g and 8 + g of 16; it
// receives the scores of head g with tokens 2r, 2r + 1, 8 + 2r, 9 + 2r.  Values O = P V: weights of just these tokens are its
// operand of P, and its operand of V is 16 (or 8) bytes of the same four tokens, two tokens' values interleaved by byte permutes.
//
// A tile of 8 heads has its upper terms in rows g and the next ones in rows g + 8, and bf16's lowest terms take a product of
// their own.  A bf16 tile of 4 heads fits all three in one product: rows h, 4 + h and 8 + h.
template <int DTYPE, int DP, int HT, bool PACKED>
struct TensorWarp {
    static constexpr int HEADS = HT;
    static constexpr bool THREE = HT == 4;       // three terms in one product
    static_assert(HT == 8 || (HT == 4 && DTYPE == TE_KV_BF16), "tiles of 8 heads, or of 4 in bf16");
    static constexpr bool E4M3 = DTYPE == TE_KV_E4M3;
    static constexpr int ES = E4M3 ? 1 : 2;
    static constexpr int TOKENS = DP * ES <= 128 ? 32 : 16;             // 8 KB a stage (16 for bf16 rows of 256)
    static constexpr int NK = TOKENS / 16;
    static constexpr int BLOCKS = blocks_per_sm(DTYPE, DP, HT);
    typedef Ring<DP, ES, TOKENS, BLOCKS == 3 ? 2 : 3, E4M3, PACKED> R;
    static constexpr int KG = E4M3 ? DP / 64 : DP / 32;                 // groups of 4 lanes x 16 bytes of a key
    static constexpr int VW = E4M3 && DP < 128 ? 8 : 16;                // bytes of a value a lane holds per chunk
    static constexpr int VE = VW / ES;                                  // elements of it
    static constexpr int VC = DP / (8 * VE);                            // chunks of 8 lanes
    static constexpr int KQ = THREE ? 2 : 4;                            // left operands of Q per group, 16 bytes a lane each
    static constexpr int Q_BYTES = KG * KQ * 32 * 16;
    static constexpr float LIFT = 10.0f;        // e4m3: weights reach 2^10, so that the lower of their two half terms keeps 2^-34 of the largest

    static constexpr int QH = HEADS / WARPS, QP = DP / 64;               // heads a warp splits, pairs of elements a lane

    // Queries into registers ahead of split_queries: heads warp, warp + 4 of the tile, lane's pairs of elements.
    struct Queries {
        float x[QH][QP][2];
    };
    static __device__ __forceinline__ void load_queries(Queries& w, const AttnParams& p, int row, const Heads& heads) {
        const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
#pragma unroll
        for (int i = 0; i < QH; ++i) {
            const int h = warp + WARPS * i;
            const float* q = p.q + row * p.qs[0] + (heads.head0 + h) * p.qs[1];
#pragma unroll
            for (int k = 0; k < QP; ++k) {
                const int c = 2 * (lane + 32 * k);
                const bool there = h < heads.count && c < p.d;
                w.x[i][k][0] = there ? q[c] : 0.0f;
                w.x[i][k][1] = there ? q[c + 1] : 0.0f;
            }
        }
    }
    // Splits them into terms, in the order the left operand wants: {row g, row g + 8, row g, row g + 8} of pairs 2j, 2j, 2j + 1, 2j + 1
    // of a lane's 16 bytes.  e4m3: operand j of 4 holds upper and lower terms of the query, brought to below 2^13 by a power of two that
    // q_unit keeps.  bf16: operand j of 2 holds upper and middle terms, operand 2 + j lower ones (and zeros in row g + 8); a tile of 4
    // heads has upper terms in rows h, middle ones in 4 + h, lower ones in 8 + h.
    static __device__ __forceinline__ void split_queries(const Queries& w, unsigned* words, float* q_unit) {
        const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
#pragma unroll
        for (int i = 0; i < QH; ++i) {
            const int h = warp + WARPS * i;
            float unit = 1.0f;
            if constexpr (E4M3) {
                float top = 0.0f;
#pragma unroll
                for (int k = 0; k < QP; ++k) top = fmaxf(top, fmaxf(fabsf(w.x[i][k][0]), fabsf(w.x[i][k][1])));
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                int e = (int)(__float_as_uint(top) >> 23) - 126 - 13;          // top < 2^(e + 13)
                e = e < -100 ? -100 : e;
                unit = __uint_as_float((unsigned)(127 - e) << 23);
                if (lane == 0) q_unit[h] = __uint_as_float((unsigned)(127 + e) << 23);
            }
#pragma unroll
            for (int k = 0; k < QP; ++k) {
                constexpr int GROUP = E4M3 ? 64 : 32, LANE = GROUP / 4;
                const int at = 2 * (lane + 32 * k), c = at / GROUP, r = at % GROUP / LANE, j = at % LANE / 2;
                unsigned* out = words + ((c * KQ + j / 2) * 32 + 4 * h + r) * 4 + j % 2 * 2;
                float x = w.x[i][k][0] * unit, y = w.x[i][k][1] * unit;
                if constexpr (E4M3) {
                    const unsigned upper = pack_half(x, y);
                    const float2 f = unpack_half(upper);
                    out[0] = upper;
                    out[1] = pack_half(x - f.x, y - f.y);
                } else {
                    const unsigned upper = pack_bf16(x, y);
                    x -= bf16_lo(upper);
                    y -= bf16_hi(upper);
                    const unsigned middle = pack_bf16(x, y), lower = pack_bf16(x - bf16_lo(middle), y - bf16_hi(middle));
                    out[0] = upper;
                    if constexpr (THREE) {
                        out[1] = lower;
                        out[4 * 4 * 4] = middle;        // four rows on: 4 x 4 lanes
                        out[4 * 4 * 4 + 1] = 0u;
                    } else {
                        out[1] = middle;
                        out[2 * 32 * 4] = lower;
                        out[2 * 32 * 4 + 1] = 0u;
                    }
                }
            }
        }
    }

    unsigned long long acc[VC * VE];     // [n tile]: 2 columns of head g, both rows of its terms
    float m, l;                // of head g; l over this lane's tokens only
    float mv;                  // e4m3: the maximum the values' weights are measured against
    float unit;                // what a score is multiplied by
    int width;                 // d: !PACKED products behind it are left out

    // The tensor core truncates as it adds to its accumulator, which over many tokens would shrink the sums; so each 16 tokens'
    // product starts from zero and is added here, rounded to nearest, with the rescaling in the same FMA.
    __device__ __forceinline__ void add(int i, const float (&x)[4], unsigned long long keep) {
        unsigned long long sum = add2(pair(x[0], x[1]), pair(x[2], x[3]));
        fma2(sum, acc[i], keep);
        acc[i] = sum;
    }

    __device__ __forceinline__ void begin(const AttnParams& p, const float* q_unit) {
#pragma unroll
        for (int i = 0; i < VC * VE; ++i) acc[i] = 0ull;
        m = mv = -INFINITY;
        l = 0.0f;
        unit = p.scale * LOG2E * (E4M3 ? q_unit[threadIdx.x % 32 / 4] : 1.0f);
        width = p.d;
    }

    // One stage's tokens, those of the bits of `seen`.
    __device__ __forceinline__ void step(const char* keys, unsigned seen, const unsigned* words) {
        const int lane = threadIdx.x % 32, g = lane / 4, r = lane % 4;
        const char* values = keys + R::SIDE;
        const float* scales = reinterpret_cast<const float*>(keys + 2 * R::SIDE);
        // ---- scores
        // (two chains of products for every 8 tokens: a product waits for the one before it in its chain)
        float sc[2 * NK][2][4];
#pragma unroll
        for (int c = 0; c < KG; ++c) {
            if (!PACKED && c > 0 && c * (4 * 16 / ES) >= width) break;
            const uint4* q = reinterpret_cast<const uint4*>(words) + c * KQ * 32 + lane;
            uint4 qw[KQ];
#pragma unroll
            for (int i = 0; i < KQ; ++i) qw[i] = q[32 * i];
#pragma unroll
            for (int i = 0; i < 2 * NK; ++i) {
                const uint4 x = *reinterpret_cast<const uint4*>(keys + R::key_at(i * 8 + g, 4 * c + r));
                float (&y)[4] = sc[i][0], (&z)[4] = sc[i][1];
                if constexpr (E4M3) {
                    const uint2 k0 = halves_of_e4m3(x.x), k1 = halves_of_e4m3(x.y), k2 = halves_of_e4m3(x.z), k3 = halves_of_e4m3(x.w);
                    mma_first_or_next<true>(c == 0, y, qw[0], k0.x, k0.y);
                    mma_first_or_next<true>(c == 0, z, qw[1], k1.x, k1.y);
                    mma<true>(y, qw[2], k2.x, k2.y);
                    mma<true>(z, qw[3], k3.x, k3.y);
                } else {
                    mma_first_or_next<false>(c == 0, y, qw[0], x.x, x.y);
                    mma_first_or_next<false>(c == 0, z, qw[1], x.z, x.w);
                    if constexpr (!THREE) {
                        mma<false>(y, qw[2], x.x, x.y);
                        mma<false>(z, qw[3], x.z, x.w);
                    }
                }
            }
        }
        float w[NK][4], vs[NK][4];
        float top = -INFINITY, topv = -INFINITY;
#pragma unroll
        for (int i = 0; i < 2 * NK; ++i) {
            const float (&y)[4] = sc[i][0], (&z)[4] = sc[i][1];
            float2 x = unpair(add2(add2(pair(y[0], y[1]), pair(z[0], z[1])), add2(pair(y[2], y[3]), pair(z[2], z[3]))));
            if constexpr (THREE) {
                x.x += __shfl_xor_sync(0xffffffffu, x.x, 16);
                x.y += __shfl_xor_sync(0xffffffffu, x.y, 16);
            }
            x.x *= unit;
            x.y *= unit;
            if constexpr (E4M3) {
                const float2 k = *reinterpret_cast<const float2*>(scales + 8 * i + 2 * r);
                x.x *= k.x;
                x.y *= k.y;
            }
            w[i / 2][i % 2 * 2] = x.x;
            w[i / 2][i % 2 * 2 + 1] = x.y;
        }
        if (seen != 0xffffffffu >> (32 - TOKENS)) {
#pragma unroll
            for (int i = 0; i < 4 * NK; ++i) w[i / 4][i % 4] = seen >> (i / 2 * 8 + 2 * r + i % 2) & 1u ? w[i / 4][i % 4] : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 4 * NK; ++i) {
            top = fmaxf(top, w[i / 4][i % 4]);
            if constexpr (E4M3) {           // a value's scale goes into its weight: 2^e, e from the exponent field
                vs[i / 4][i % 4] = w[i / 4][i % 4] + (float)((int)(__float_as_uint(scales[TOKENS + i / 2 * 8 + 2 * r + i % 2]) >> 23) - 127);
                topv = fmaxf(topv, vs[i / 4][i % 4]);
            }
        }
        // ---- weights
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        top = fmaxf(top, m);
        const float base = settled(top);
        float keep = exp2_of(m - base), sum = 0.0f;
#pragma unroll
        for (int nk = 0; nk < NK; ++nk)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = exp2_of(w[nk][i] - base);
                sum += e;
                if constexpr (!E4M3) w[nk][i] = e;
            }
        l = l * keep + sum;
        m = top;
        if constexpr (E4M3) {
            topv = fmaxf(topv, __shfl_xor_sync(0xffffffffu, topv, 1));
            topv = fmaxf(topv, __shfl_xor_sync(0xffffffffu, topv, 2));
            topv = fmaxf(topv, mv);
            const float basev = settled(topv);
            keep = exp2_of(mv - basev);
#pragma unroll
            for (int nk = 0; nk < NK; ++nk)
#pragma unroll
                for (int i = 0; i < 4; ++i) w[nk][i] = exp2_of(vs[nk][i] - basev + LIFT);
            mv = topv;
        }
        uint4 a[NK], lower[NK];         // left operands of P; bf16: the lowest terms apart
#pragma unroll
        for (int nk = 0; nk < NK; ++nk) {
            float x0 = w[nk][0], x1 = w[nk][1], x2 = w[nk][2], x3 = w[nk][3];
            if constexpr (E4M3) {
                a[nk].x = pack_half(x0, x1);
                a[nk].z = pack_half(x2, x3);
                const float2 f = unpack_half(a[nk].x), h = unpack_half(a[nk].z);
                a[nk].y = pack_half(x0 - f.x, x1 - f.y);
                a[nk].w = pack_half(x2 - h.x, x3 - h.y);
            } else {
                a[nk].x = pack_bf16(x0, x1);
                a[nk].z = pack_bf16(x2, x3);
                x0 -= bf16_lo(a[nk].x); x1 -= bf16_hi(a[nk].x); x2 -= bf16_lo(a[nk].z); x3 -= bf16_hi(a[nk].z);
                a[nk].y = pack_bf16(x0, x1);
                a[nk].w = pack_bf16(x2, x3);
                lower[nk] = make_uint4(pack_bf16(x0 - bf16_lo(a[nk].y), x1 - bf16_hi(a[nk].y)), 0u, pack_bf16(x2 - bf16_lo(a[nk].w), x3 - bf16_hi(a[nk].w)), 0u);
                if constexpr (THREE) {      // heads' lanes hold upper and lower terms, the other half middle ones
                    a[nk] = g < 4 ? make_uint4(a[nk].x, lower[nk].x, a[nk].z, lower[nk].z) : make_uint4(a[nk].y, 0u, a[nk].w, 0u);
                }
            }
        }
        // ---- values
        const unsigned long long keep2 = pair(keep, keep);
#pragma unroll
        for (int c = 0; c < VC; ++c) {
            if (!PACKED && c > 0 && c * 8 * VE >= width) break;
            unsigned x[NK][4][4];
#pragma unroll
            for (int nk = 0; nk < NK; ++nk)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = nk * 16 + 8 * (i / 2) + 2 * r + i % 2;
                    if constexpr (VW == 16) {
                        const uint4 v = *reinterpret_cast<const uint4*>(values + R::value_at(t, 8 * c + g));
                        x[nk][i][0] = v.x; x[nk][i][1] = v.y; x[nk][i][2] = v.z; x[nk][i][3] = v.w;
                    } else {
                        const uint2 v = *reinterpret_cast<const uint2*>(values + R::value_at(t, 4 * c + g / 2) + g % 2 * 8);
                        x[nk][i][0] = v.x; x[nk][i][1] = v.y;
                    }
                }
#pragma unroll
            for (int i = 0; i < VW / 4; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float y0[4], y1[4];
#pragma unroll
                    for (int nk = 0; nk < NK; ++nk) {
                        if constexpr (E4M3) {
                            const uint2 b0 = halves_of_e4m3(__byte_perm(x[nk][0][i], x[nk][1][i], e ? 0x7362 : 0x5140));
                            const uint2 b1 = halves_of_e4m3(__byte_perm(x[nk][2][i], x[nk][3][i], e ? 0x7362 : 0x5140));
                            if (nk == 0) mma_from_zero<true>(y0, a[nk], b0.x, b1.x);
                            else mma<true>(y0, a[nk], b0.x, b1.x);
                            if (nk == 0) mma_from_zero<true>(y1, a[nk], b0.y, b1.y);
                            else mma<true>(y1, a[nk], b0.y, b1.y);
                        } else {
                            const unsigned b0 = __byte_perm(x[nk][0][i], x[nk][1][i], e ? 0x7632 : 0x5410), b1 = __byte_perm(x[nk][2][i], x[nk][3][i], e ? 0x7632 : 0x5410);
                            if (nk == 0) mma_from_zero<false>(y0, a[nk], b0, b1);
                            else mma<false>(y0, a[nk], b0, b1);
                            if constexpr (!THREE) mma<false>(y0, lower[nk], b0, b1);
                        }
                    }
                    if constexpr (E4M3) {
                        add(c * VE + 4 * i + 2 * e, y0, keep2);
                        add(c * VE + 4 * i + 2 * e + 1, y1, keep2);
                    } else {
                        add(c * VE + 2 * i + e, y0, keep2);
                    }
                }
        }
    }

    // What is left to do when the last stage has been seen.
    __device__ __forceinline__ void finish() {
        // one sum per head, and e4m3 sums measured against m like the others
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const float back = E4M3 ? exp2_of(settled(mv) - settled(m) - LIFT) : 1.0f;
#pragma unroll
        for (int i = 0; i < VC * VE; ++i) {
            if constexpr (E4M3) acc[i] = mul2(acc[i], pair(back, back));
            if constexpr (THREE) {
                const float2 x = unpair(acc[i]);
                acc[i] = pair(x.x + __shfl_xor_sync(0xffffffffu, x.x, 16), x.y + __shfl_xor_sync(0xffffffffu, x.y, 16));
            }
        }
    }

    // This warp's sums into shared memory: acc [HEADS][DP], ml [HEADS].
    __device__ __forceinline__ void put(float* out, float2* ml) const {
        const int lane = threadIdx.x % 32, g = lane / 4, r = lane % 4;
        if (g >= HEADS) return;
        if (r == 0) ml[g] = make_float2(m, l);
#pragma unroll
        for (int c = 0; c < VC; ++c)
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                float* at = out + g * DP + c * 8 * VE + 2 * r * VE + j;
                const float2 x = unpair(acc[c * VE + j]);
                at[0] = x.x;
                at[VE] = x.y;
            }
    }
};

// ------------------------------------------------------------------------------------------------------ FP32 cache
// One warp's share of a segment with FP32 FMAs, HT heads at once.  Scores: lane (g, r) takes 16-byte pieces r, r + 4, .. of
// token g's key (and of token 8 + g's), and four lanes add up to a score.  Values: the lanes lie along d, and the weights
// come back through a few words of shared memory.
template <int DP, int HT, bool PACKED>
struct FmaWarp {
    static constexpr int HEADS = HT;
    static constexpr int TOKENS = DP <= 64 ? 16 : 8;
    static constexpr int BLOCKS = blocks_per_sm(TE_KV_F32, DP, HT);
    typedef Ring<DP, 4, TOKENS, BLOCKS == 3 ? 2 : 3, false, PACKED> R;
    static constexpr int TG = TOKENS / 8;                  // tokens whose keys a lane takes parts of
    static constexpr int KC = DP / 16;                     // 16-byte pieces of a key a lane takes
    static constexpr int LPT = DP / 4 < 32 ? DP / 4 : 32;  // lanes along a value
    static constexpr int TPI = 32 / LPT;                   // tokens the warp takes at once
    static constexpr int VC = DP / 4 / LPT;                // pieces of a value a lane takes
    static constexpr int VI = TOKENS / TPI;
    static constexpr int OWN = (HT + 3) / 4;               // heads whose weights a lane computes
    static constexpr int Q_BYTES = HT * DP * 4 + WARPS * (TOKENS * HT + HT) * 8;     // queries, then each warp's weights and factors,
                                                                                     // doubled for two FMAs at once

    static constexpr int QN = (HT * DP + THREADS - 1) / THREADS;

    struct Queries {
        float x[QN];
    };
    static __device__ __forceinline__ void load_queries(Queries& w, const AttnParams& p, int row, const Heads& heads) {
        const float* q = p.q + row * p.qs[0] + heads.head0 * p.qs[1];
#pragma unroll
        for (int k = 0; k < QN; ++k) {
            const int i = threadIdx.x + k * THREADS, h = i / DP, c = i % DP;
            w.x[k] = h < heads.count && c < p.d ? q[h * p.qs[1] + c] : 0.0f;
        }
    }
    static __device__ __forceinline__ void split_queries(const Queries& w, unsigned* words, float*) {
#pragma unroll
        for (int k = 0; k < QN; ++k) {
            const int i = threadIdx.x + k * THREADS;
            if (i < HT * DP) reinterpret_cast<float*>(words)[i] = w.x[k];
        }
    }

    unsigned long long acc[HT][VC][2];
    float m[OWN], l[OWN];          // of heads r, r + 4 (modulo HT); l over this lane's tokens only

    float unit;                    // what a score is multiplied by
    int width;                     // d: !PACKED pieces behind it are left out

    __device__ __forceinline__ void begin(const AttnParams& p, const float*) {
#pragma unroll
        for (int h = 0; h < HT; ++h)
#pragma unroll
            for (int c = 0; c < VC; ++c) acc[h][c][0] = acc[h][c][1] = 0ull;
#pragma unroll
        for (int i = 0; i < OWN; ++i) { m[i] = -INFINITY; l[i] = 0.0f; }
        unit = p.scale * LOG2E;
        width = p.d;
    }

    __device__ __forceinline__ void step(const char* keys, unsigned seen, unsigned* words) {
        const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, r = lane % 4;
        const int along = lane % LPT, which = lane / LPT;
        const char* values = keys + R::SIDE;
        const float* q = reinterpret_cast<const float*>(words);
        unsigned long long* weights = reinterpret_cast<unsigned long long*>(words + HT * DP) + warp * (TOKENS * HT + HT);
        unsigned long long* factors = weights + TOKENS * HT;
        // ---- scores: every lane of a quad ends with the sums of all heads
        float sc[TG][HT];
#pragma unroll
        for (int i = 0; i < TG; ++i) {
            unsigned long long part[HT][2];
#pragma unroll
            for (int h = 0; h < HT; ++h) part[h][0] = part[h][1] = 0ull;
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                if (!PACKED && c * 16 >= width) break;
                const ulonglong2 kk = *reinterpret_cast<const ulonglong2*>(keys + R::key_at(g + 8 * i, 4 * c + r));
#pragma unroll
                for (int h = 0; h < HT; ++h) {
                    const ulonglong2 qq = *reinterpret_cast<const ulonglong2*>(q + h * DP + c * 16 + r * 4);
                    fma2(part[h][0], qq.x, kk.x);
                    fma2(part[h][1], qq.y, kk.y);
                }
            }
#pragma unroll
            for (int h = 0; h < HT; ++h) {
                const float2 x = unpair(part[h][0]), y = unpair(part[h][1]);
                sc[i][h] = (x.x + x.y) + (y.x + y.y);
                sc[i][h] += __shfl_xor_sync(0xffffffffu, sc[i][h], 1);
                sc[i][h] += __shfl_xor_sync(0xffffffffu, sc[i][h], 2);
            }
        }
        // ---- weights of heads r, r + 4 over tokens g (and 8 + g)
        bool moved = false;
#pragma unroll
        for (int j = 0; j < OWN; ++j) {
            const int h = (r + 4 * j) % HT;
            float w[TG], top = m[j];
#pragma unroll
            for (int i = 0; i < TG; ++i) {
                float x = sc[i][(4 * j) % HT];
#pragma unroll
                for (int u = 1; u < 4; ++u) x = r == u ? sc[i][(u + 4 * j) % HT] : x;
                w[i] = seen >> (g + 8 * i) & 1u ? x * unit : -INFINITY;
                top = fmaxf(top, w[i]);
            }
#pragma unroll
            for (int o = 4; o < 32; o *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float base = settled(top), keep = exp2_of(m[j] - base);
            l[j] *= keep;
            moved |= top != m[j];
            m[j] = top;
#pragma unroll
            for (int i = 0; i < TG; ++i) {
                const float e = exp2_of(w[i] - base);
                l[j] += e;
                weights[(g + 8 * i) * HT + h] = pair(e, e);
            }
            if (g == 0) factors[h] = pair(keep, keep);
        }
        moved = __any_sync(0xffffffffu, moved);
        __syncwarp();
        if (moved) {
#pragma unroll
            for (int h = 0; h < HT; ++h) {
                const unsigned long long f = factors[h];
#pragma unroll
                for (int c = 0; c < VC; ++c) {
                    acc[h][c][0] = mul2(acc[h][c][0], f);
                    acc[h][c][1] = mul2(acc[h][c][1], f);
                }
            }
        }
        // ---- values
#pragma unroll
        for (int i = 0; i < VI; ++i) {
            const int t = i * TPI + which;
            const unsigned long long* w = weights + t * HT;
#pragma unroll
            for (int c = 0; c < VC; ++c) {
                const ulonglong2 vv = *reinterpret_cast<const ulonglong2*>(values + R::value_at(t, c * 32 + along));
#pragma unroll
                for (int h = 0; h < HT; ++h) {
                    const unsigned long long x = w[h];
                    fma2(acc[h][c][0], x, vv.x);
                    fma2(acc[h][c][1], x, vv.y);
                }
            }
        }
        __syncwarp();                  // the weights have been read
    }

    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int j = 0; j < OWN; ++j)
#pragma unroll
            for (int o = 4; o < 32; o *= 2) l[j] += __shfl_xor_sync(0xffffffffu, l[j], o);
        // lanes that hold other tokens of the same elements
#pragma unroll
        for (int o = LPT; o < 32; o *= 2)
#pragma unroll
            for (int h = 0; h < HT; ++h)
#pragma unroll
                for (int c = 0; c < VC; ++c)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float2 x = unpair(acc[h][c][i]);
                        acc[h][c][i] = pair(x.x + __shfl_xor_sync(0xffffffffu, x.x, o), x.y + __shfl_xor_sync(0xffffffffu, x.y, o));
                    }
    }

    __device__ __forceinline__ void put(float* out, float2* ml) const {
        const int lane = threadIdx.x % 32, g = lane / 4, r = lane % 4;
#pragma unroll
        for (int j = 0; j < OWN; ++j)
            if (g == 0 && r + 4 * j < HT) ml[r + 4 * j] = make_float2(m[j], l[j]);
        if (lane < LPT) {
#pragma unroll
            for (int h = 0; h < HT; ++h)
#pragma unroll
                for (int c = 0; c < VC; ++c) {
                    ulonglong2 x;
                    x.x = acc[h][c][0];
                    x.y = acc[h][c][1];
                    *reinterpret_cast<ulonglong2*>(out + h * DP + c * 128 + lane * 4) = x;
                }
        }
    }
};

template <int DTYPE, int DP, int HT, bool PACKED> struct WarpOf { typedef TensorWarp<DTYPE, DP, HT, PACKED> type; };
template <int DP, int HT, bool PACKED> struct WarpOf<TE_KV_F32, DP, HT, PACKED> { typedef FmaWarp<DP, HT, PACKED> type; };

// ---------------------------------------------------------------------------------------------------- the two kernels
// Four elements of a head's result, from its sums.
__device__ __forceinline__ void put_result(const AttnParams& p, int row, int head, int c, const float4& a, float m, float l) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    float* o = p.o + row * p.os[0] + head * p.os[1] + c;
    o[0] = a.x * inv; o[1] = a.y * inv; o[2] = a.z * inv; o[3] = a.w * inv;
    if (p.lse && c == 0) p.lse[(int64_t)row * p.q_heads + head] = l == 0.0f ? -INFINITY : (m + log2f(l)) * LN2;
}

template <int DTYPE, int DP, int HT, bool PACKED>
__global__ void __launch_bounds__(THREADS, WarpOf<DTYPE, DP, HT, PACKED>::type::BLOCKS) paged_attention_kernel(const AttnParams p) {
    typedef typename WarpOf<DTYPE, DP, HT, PACKED>::type Warp;
    typedef typename Warp::R R;
    constexpr int HEADS = Warp::HEADS, TILE = R::STEP;
    extern __shared__ __align__(128) char shared[];
    char* rings = shared;                                  // [WARPS][R::BYTES]
    unsigned* query = reinterpret_cast<unsigned*>(shared + WARPS * R::BYTES);       // [Warp::Q_BYTES]
    static_assert(HEADS * DP * 4 <= R::STAGE, "a warp's sums fit the stage it read last");
    __shared__ float2 ml[WARPS][HEADS];
    __shared__ float q_unit[HEADS];
    __shared__ int scan[WARPS];
    __shared__ int found_prefix;
    __shared__ int found_row;
    __shared__ bool last_part;
    griddep_wait();
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    const int w = blockIdx.x;
    const int tiles_of_heads = p.kv_heads * p.head_tiles;
    auto range_of = [&](int r) { return row_range(p.lens[r], p.most, p.window); };

    // ---- this worker's share: the rows' units, added up by all threads over slabs of rows
    const int slab = (p.rows + THREADS - 1) / THREADS;
    const int r0 = min(p.rows, tid * slab), r1 = min(p.rows, r0 + slab);
    int mine = 0;
    bool cut = false, empty = false;
    for (int r = r0; r < r1; ++r) {
        const int64_t len = p.lens[r];
        cut |= len > p.most;
        const int c = segment_units(row_tiles(row_range(len, p.most, p.window), TILE));
        empty |= c == 0;
        mine += c;
    }
    if (cut) atomicCAS(p.status, 0, STATUS_BAD_CACHE_PLACE);
    int before = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int x = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += x;
    }
    if (lane == 31) scan[warp] = before;
    empty = __syncthreads_or(empty);
    int total = 0;
    before -= mine;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
        if (i < warp) before += scan[i];
        total += scan[i];
    }
    const int units = total * tiles_of_heads;
    // every worker has a unit; on the tensor cores two, since a part costs a join (32768 tokens of one key head: 21 us against
    // 26 with one; with four, eight rows of 1024 tokens or less take 12 us against 10)
    const Shares shares = shares_of(units, max(1, min(units / (DTYPE == TE_KV_F32 ? 1 : 2), (int)gridDim.x)));
    const int unit = w < shares.workers ? share_begin(shares, w) : 0;
    const int unit_end = w < shares.workers ? share_begin(shares, w + 1) : 0;
    if (unit < unit_end) {
        const int at = (int)((unsigned)unit / (unsigned)tiles_of_heads);          // in the rows' sums
        if (at >= before && at < before + mine) {
            for (int r = r0; r < r1; ++r) {
                const int c = r1 - r0 == 1 ? mine : segment_units(row_tiles(range_of(r), TILE));
                if (at < before + c) {
                    found_row = r;
                    found_prefix = before;
                    break;
                }
                before += c;
            }
        }
    }
    if (tid == 0 && !p.arrived) p.joins[w] = make_int4(0, 0, 0, 0);
    __syncthreads();
    if (empty) {        // some row without tokens
        for (int r = w; r < p.rows; r += gridDim.x) {
            if (row_tiles(range_of(r), TILE) > 0) continue;
            for (int i = tid; i < p.q_heads * p.d; i += THREADS) p.o[r * p.os[0] + i / p.d * p.os[1] + i % p.d] = 0.0f;
            if (p.lse)
                for (int i = tid; i < p.q_heads; i += THREADS) p.lse[(int64_t)r * p.q_heads + i] = -INFINITY;
        }
    }
    if (unit >= unit_end) return;

    // ---- its pieces of segments.  Copies run ahead of the arithmetic, into the next pieces as well, so each side
    // goes through the pieces by itself.
    Walker behind;
    behind.start(unit, unit_end, found_row, found_prefix * tiles_of_heads);
    Walker ahead = behind;
    Piece piece, soon;
    if (!behind.next(range_of, tiles_of_heads, TILE, piece)) return;        // a share that lies in a segment's SEGMENT_COST
    ahead.next(range_of, tiles_of_heads, TILE, soon);
    char* ring = rings + warp * R::BYTES;
    R copies;
    copies.base = smem_address(ring);
    int soon_head = heads_of<HEADS>(p, soon.head_tile).kv_head;
    int t0 = soon.first_tile * TILE + warp * R::TOKENS;                      // of this warp's next stage
    copies.look_up(p, p.page_table + soon.row * p.table_stride, t0, soon.range.n);
    auto issue_next = [&](int stage) {
        unsigned seen = 0u;
        if (soon.tiles > 0) {
            seen = copies.issue(p, soon.range, soon_head, t0, stage);
            t0 += TILE;
            if (--soon.tiles == 0 && ahead.next(range_of, tiles_of_heads, TILE, soon)) {
                t0 = soon.first_tile * TILE + warp * R::TOKENS;
                soon_head = heads_of<HEADS>(p, soon.head_tile).kv_head;
            }
            if (soon.tiles > 0) copies.look_up(p, p.page_table + soon.row * p.table_stride, t0, soon.range.n);
        }
        copies_issued();
        return seen;
    };
    Heads heads = heads_of<HEADS>(p, piece.head_tile);
    typename Warp::Queries loaded;
    Warp::load_queries(loaded, p, piece.row, heads);
    unsigned seen[R::STAGES];           // of the stages under way, the next to be read first
#pragma unroll
    for (int i = 0; i < R::STAGES - 1; ++i) seen[i] = issue_next(i);
    Warp::split_queries(loaded, query, q_unit);
    __syncthreads();
    int at = 0, to = R::STAGES - 1;
    for (;;) {
        Warp sums_here;
        sums_here.begin(p, q_unit);
        for (int n = 0; n < piece.tiles; ++n) {
            copies_wait<R::STAGES - 2>();
            __syncwarp();               // this stage has landed for all lanes, and all are done with the one before it
            seen[R::STAGES - 1] = issue_next(to);
            sums_here.step(ring + at * R::STAGE, seen[0], query);
#pragma unroll
            for (int i = 0; i + 1 < R::STAGES; ++i) seen[i] = seen[i + 1];
            at = at + 1 == R::STAGES ? 0 : at + 1;
            to = to + 1 == R::STAGES ? 0 : to + 1;
        }
        Piece next = piece;
        const bool more = behind.next(range_of, tiles_of_heads, TILE, next);
        const Heads next_heads = heads_of<HEADS>(p, next.head_tile);
        if (more) Warp::load_queries(loaded, p, next.row, next_heads);
        sums_here.finish();
        __syncwarp();
        // no copy is under way into the stage read last, which is the next to be filled
        auto sums = [&](int j, int h, int c) { return reinterpret_cast<float*>(rings + j * R::BYTES + to * R::STAGE) + h * DP + c; };
        sums_here.put(sums(warp, 0, 0), ml[warp]);
        __syncthreads();
        // ---- the four warps' sums into the result, or into the workspace when the segment is shared with other workers
        const bool whole = piece.begins && piece.ends;
        const int slot = part_slot(w, piece.begins);
        for (int i = tid; i < heads.count * (DP / 4); i += THREADS) {
            const int h = i / (DP / 4), c = i % (DP / 4) * 4;
            if (c >= p.d) continue;
            float m = ml[0][h].x;
#pragma unroll
            for (int j = 1; j < WARPS; ++j) m = fmaxf(m, ml[j][h].x);
            const float base = settled(m);
            float l = 0.0f;
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int j = 0; j < WARPS; ++j) {
                const float f = exp2_of(ml[j][h].x - base);
                const float4 x = *reinterpret_cast<const float4*>(sums(j, h, c));
                l += f * ml[j][h].y;
                a.x += f * x.x; a.y += f * x.y; a.z += f * x.z; a.w += f * x.w;
            }
            if (whole) {
                put_result(p, piece.row, heads.head0 + h, c, a, m, l);
            } else {
                *reinterpret_cast<float4*>(p.part_acc + ((int64_t)slot * HEADS + h) * p.d + c) = a;
                if (c == 0) p.part_ml[slot * HEADS + h] = make_float2(m, l);
            }
        }
        if (!whole && p.arrived) {
            // whoever finishes a segment's last part adds them all, in the order of the tokens
            const int tiles = row_tiles(piece.range, TILE);
            const int first = worker_of(shares, piece.segment_end - tiles), parts = worker_of(shares, piece.segment_end - 1) - first + 1;
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                last_part = atomicAdd(p.arrived + first, 1) == parts - 1;
                if (last_part) p.arrived[first] = 0;
            }
            __syncthreads();
            if (last_part) {
                __threadfence();
                for (int i = tid; i < heads.count * (DP / 4); i += THREADS) {
                    const int h = i / (DP / 4), c = i % (DP / 4) * 4;
                    if (c >= p.d) continue;
                    auto place = [&](int k) { return (int64_t)part_slot(first + k, k == 0) * HEADS + h; };
                    float m = -INFINITY;
#pragma unroll 4
                    for (int k = 0; k < parts; ++k) m = fmaxf(m, __ldcg(p.part_ml + place(k)).x);
                    const float base = settled(m);
                    float l = 0.0f;
                    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                    for (int k = 0; k < parts; ++k) {
                        const float2 part = __ldcg(p.part_ml + place(k));
                        const float4 x = __ldcg(reinterpret_cast<const float4*>(p.part_acc + place(k) * p.d + c));
                        const float f = exp2_of(part.x - base);
                        l += f * part.y;
                        a.x += f * x.x; a.y += f * x.y; a.z += f * x.z; a.w += f * x.w;
                    }
                    put_result(p, piece.row, heads.head0 + h, c, a, m, l);
                }
            }
        } else if (tid == 0 && piece.begins && !piece.ends) {
            p.joins[w] = make_int4(piece.row, piece.head_tile, worker_of(shares, piece.segment_end - 1), 1);
        }
        if (!more) return;
        Warp::split_queries(loaded, query, q_unit);
        __syncthreads();
        piece = next;
        heads = next_heads;
    }
}

// Adds the parts of the segment that begins in worker blockIdx.x's share, in the order of its tokens, for head blockIdx.y of
// the tile: warps take parts in turn, lanes lie along d; then the warps' sums are added in order.
constexpr int JOIN_WARPS = 16;
__global__ void __launch_bounds__(32 * JOIN_WARPS) paged_join_kernel(const AttnParams p, int heads_per_tile) {
    __shared__ float sums[JOIN_WARPS][256];
    __shared__ float tops[JOIN_WARPS], totals[JOIN_WARPS];
    griddep_wait();
    const int w = blockIdx.x, h = blockIdx.y, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int4 j = p.joins[w];
    if (!j.w) return;
    const int kv_head = j.y / p.head_tiles, part = j.y % p.head_tiles * heads_per_tile;
    if (part + h >= p.group) return;
    const int count = j.z - w + 1;
    auto at = [&](int i) { return (int64_t)part_slot(w + i, i == 0) * heads_per_tile + h; };
    float m = -INFINITY;
    for (int i = threadIdx.x; i < count; i += 32 * JOIN_WARPS) m = fmaxf(m, p.part_ml[at(i)].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) tops[warp] = m;
    __syncthreads();
    m = tops[0];
#pragma unroll
    for (int i = 1; i < JOIN_WARPS; ++i) m = fmaxf(m, tops[i]);
    const float base = settled(m);
    float a[8] = {}, l = 0.0f;
#pragma unroll 8
    for (int i = warp; i < count; i += JOIN_WARPS) {
        const int64_t o = at(i);
        const float2 ml = p.part_ml[o];
        const float f = exp2_of(ml.x - base);
        l += f * ml.y;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int c = u * 128 + lane * 4;
            if (c < p.d) {
                const float4 x = *reinterpret_cast<const float4*>(p.part_acc + o * p.d + c);
                a[4 * u] += f * x.x; a[4 * u + 1] += f * x.y; a[4 * u + 2] += f * x.z; a[4 * u + 3] += f * x.w;
            }
        }
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) sums[warp][u / 4 * 128 + lane * 4 + u % 4] = a[u];
    if (lane == 0) totals[warp] = l;
    __syncthreads();
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < JOIN_WARPS; ++i) l += totals[i];
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int head = kv_head * p.group + part + h;
    for (int c = threadIdx.x; c < p.d; c += 32 * JOIN_WARPS) {
        float x = 0.0f;
#pragma unroll
        for (int i = 0; i < JOIN_WARPS; ++i) x += sums[i][c];
        p.o[j.x * p.os[0] + head * p.os[1] + c] = x * inv;
    }
    if (p.lse && threadIdx.x == 0) p.lse[(int64_t)j.x * p.q_heads + head] = l == 0.0f ? -INFINITY : (m + log2f(l)) * LN2;
}

// ------------------------------------------------------------------------------------------------------------ host side
// Heads a tile holds.  Every head of a tile is computed whether it is there or not, so: with FMAs the smallest of 1, 2, 4, 8
// that takes the group; on the tensor cores 4 where that takes it in bf16, which halves the products (16 rows of 20 key heads
// with one query head each, window 4096: 40 us against 46 with tiles of 8), else 8.
int heads_per_tile(int dtype, int64_t group) {
    if (dtype == TE_KV_E4M3 || group >= 5) return 8;
    return dtype == TE_KV_BF16 || group >= 3 ? 4 : (int)group;
}

size_t workspace_need(const te_paged_attn_desc* t, int sm_count) {
    if (t->rows == 0 || t->q_heads == 0) return 0;
    const int tile = heads_per_tile(t->cache.dtype, t->q_heads / t->cache.heads);
    const size_t workers = (size_t)sm_count * blocks_per_sm(t->cache.dtype, (int)t->cache.d, tile), heads = tile;
    return workers * 16 + 2 * workers * heads * (8 + 4 * (size_t)t->cache.d);
}

template <int DTYPE, int DP, int HT, bool PACKED>
cudaError_t launch_form(te_b200_ctx* ctx, const AttnParams& p, int workers, cudaStream_t st) {
    typedef typename WarpOf<DTYPE, DP, HT, PACKED>::type Warp;
    auto kernel = paged_attention_kernel<DTYPE, DP, HT, PACKED>;
    constexpr int bytes = WARPS * Warp::R::BYTES + Warp::Q_BYTES;
    int& state = ctx->kernel_state[reinterpret_cast<const void*>(kernel)];
    if (!state) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != cudaSuccess) return e;
        state = 1;
    }
    return launch_pdl(kernel, dim3(workers), dim3(THREADS), bytes, st, p);
}

template <int DTYPE, int DP, int HT>
cudaError_t launch_tiles(te_b200_ctx* ctx, const AttnParams& p, int workers, cudaStream_t st) {
    constexpr int64_t row = DP * (DTYPE == TE_KV_F32 ? 4 : DTYPE == TE_KV_BF16 ? 2 : 1);
    const bool packed = p.d == DP && p.page_size.divisor % 16 == 0 && p.kcs[2] == row && p.vcs[2] == row;
    return packed ? launch_form<DTYPE, DP, HT, true>(ctx, p, workers, st) : launch_form<DTYPE, DP, HT, false>(ctx, p, workers, st);
}

template <int DP>
cudaError_t launch_width(te_b200_ctx* ctx, const AttnParams& p, int dtype, int heads, int workers, cudaStream_t st) {
    if (dtype == TE_KV_BF16 && heads == 4) return launch_tiles<TE_KV_BF16, DP, 4>(ctx, p, workers, st);
    if (dtype == TE_KV_BF16) return launch_tiles<TE_KV_BF16, DP, 8>(ctx, p, workers, st);
    if (dtype == TE_KV_E4M3) return launch_tiles<TE_KV_E4M3, DP, 8>(ctx, p, workers, st);
    if (heads == 1) return launch_tiles<TE_KV_F32, DP, 1>(ctx, p, workers, st);
    if (heads == 2) return launch_tiles<TE_KV_F32, DP, 2>(ctx, p, workers, st);
    if (heads == 4) return launch_tiles<TE_KV_F32, DP, 4>(ctx, p, workers, st);
    return launch_tiles<TE_KV_F32, DP, 8>(ctx, p, workers, st);
}

int check_desc(const te_paged_attn_desc* t) {
    if (!t || t->rows < 0 || t->q_heads < 0 || t->max_pages < 0) return fail(TE_ERR_BAD_ARGUMENT, "paged attention: bad extents");
    if (int bad = check_kv_cache(t->cache, "paged attention")) return bad;
    const te_kv_cache& c = t->cache;
    if (t->q_heads > 0 && (c.heads == 0 || t->q_heads % c.heads)) return fail(TE_ERR_BAD_ARGUMENT, "paged attention: q_heads must be a multiple of the cache's heads");
    if (t->max_pages > 0 && c.page_size > (INT32_MAX - 4096) / t->max_pages) return fail(TE_ERR_BAD_ARGUMENT, "paged attention: the page table reaches beyond 2^31-1 positions");
    if (t->q_heads > 65535 || (t->q_heads > 0 && t->rows > INT32_MAX / t->q_heads)) return fail(TE_ERR_BAD_ARGUMENT, "paged attention: too many rows or heads");
    if (t->max_pages > 0 && (t->max_pages * c.page_size / 32 + 4) * t->q_heads >= INT32_MAX)
        return fail(TE_ERR_BAD_ARGUMENT, "paged attention: too many heads for so long a page table");
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
    *out_bytes = workspace_need(d, sm_count);
    return TE_OK;
}

int te_b200_paged_attention(te_b200_ctx* ctx, const te_paged_attn_desc* t, te_stream_t stream) {
    if (int bad = check_desc(t)) return bad;
    if (int bad = check_ctx(ctx)) return bad;
    if (t->rows == 0 || t->q_heads == 0) return TE_OK;
    const te_kv_cache& c = t->cache;
    const size_t need = workspace_need(t, ctx->sm_count);
    if (need > ctx->workspace_bytes) {
        char msg[160];
        snprintf(msg, sizeof msg, "context workspace (%zu bytes) too small; paged attention needs %zu bytes", ctx->workspace_bytes, need);
        return fail(TE_ERR_WORKSPACE, msg);
    }
    AttnParams p;
    p.kc = static_cast<const char*>(c.k); p.vc = static_cast<const char*>(c.v); p.k_scale = c.k_scale; p.v_scale = c.v_scale;
    const int64_t size = c.dtype == TE_KV_F32 ? 4 : c.dtype == TE_KV_BF16 ? 2 : 1;
    for (int i = 0; i < 2; ++i) { p.qs[i] = t->q_strides[i]; p.os[i] = t->o_strides[i]; }
    for (int i = 0; i < 3; ++i) { p.kcs[i] = c.k_strides[i] * size; p.vcs[i] = c.v_strides[i] * size; p.ss[i] = c.scale_strides[i]; }
    p.table_stride = t->page_table_stride; p.pages = c.pages; p.window = t->window;
    p.page_size = make_fast_divisor((uint32_t)c.page_size);
    p.most = c.pages > 0 ? (int)(t->max_pages * c.page_size) : 0;      // (a cache without pages has no places)
    p.q_heads = (int)t->q_heads; p.kv_heads = (int)c.heads;
    p.group = (int)(t->q_heads / c.heads); p.d = (int)c.d;
    const int heads = heads_per_tile(c.dtype, p.group);
    const int workers = ctx->sm_count * blocks_per_sm(c.dtype, p.d, heads);
    p.head_tiles = (p.group + heads - 1) / heads;
    p.scale = t->scale;
    char* ws = static_cast<char*>(ctx->workspace);
    p.joins = reinterpret_cast<int4*>(ws);
    p.part_ml = reinterpret_cast<float2*>(ws + (size_t)workers * 16);
    p.part_acc = reinterpret_cast<float*>(ws + (size_t)workers * 16 + (size_t)workers * 2 * heads * 8);
    p.status = ctx->d_status;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // so many rows at a time that their units stay below 2^31 (a tile has 32 tokens or more): nearly always all
    const int64_t row_units = ((int64_t)p.most / 32 + 2 + SEGMENT_COST) * p.kv_heads * p.head_tiles;
    const int64_t rows_at_once = INT32_MAX / row_units;
    for (int64_t r = 0; r < t->rows; r += rows_at_once) {
        p.rows = (int)(t->rows - r < rows_at_once ? t->rows - r : rows_at_once);
        p.q = t->q + r * t->q_strides[0];
        p.o = t->o + r * t->o_strides[0];
        p.lse = t->lse ? t->lse + r * t->q_heads : nullptr;
        p.page_table = t->page_table + r * t->page_table_stride;
        p.lens = t->lens + r;
        // Parts of a segment: at most one per tile, and on average workers per segment.  Few are added by the block that
        // finishes last, which saves a launch (32 ragged bf16 rows of 8 key heads: 86 us against 90 with the second
        // kernel); many would keep that one block busy (32768 tokens of one key head: 92 us against 21), so a kernel of
        // their own adds them.
        const int64_t segments = (int64_t)p.rows * p.kv_heads * p.head_tiles;
        int64_t parts = p.most / 32 + 1;
        if (parts > workers / segments + 1) parts = workers / segments + 1;
        const bool join_inside = parts <= 16 && workers <= STATUS_COUNTER_WORDS;
        p.arrived = join_inside ? ctx->d_status + STATUS_COUNTER_WORD : nullptr;
        cudaError_t e = p.d <= 64 ? launch_width<64>(ctx, p, c.dtype, heads, workers, st) : p.d <= 128 ? launch_width<128>(ctx, p, c.dtype, heads, workers, st)
                                                                                      : launch_width<256>(ctx, p, c.dtype, heads, workers, st);
        if (e != cudaSuccess) return cuda_fail(e, "paged_attention_kernel launch");
        ctx->launches += 1;
        if (join_inside) continue;
        e = launch_pdl(paged_join_kernel, dim3((unsigned)workers, (unsigned)heads), dim3(32 * JOIN_WARPS), 0, st, p, heads);
        if (e != cudaSuccess) return cuda_fail(e, "paged_join_kernel launch");
        ctx->launches += 1;
    }
    return TE_OK;
}

}  // extern "C"

// Attention of new tokens over the paged 4-bit cache.
//
// With value = code * s + m for a group of 32 channels,
//   q . k_t      = sum_g s_tg (q_g . c_tg) + m_tg sum(q_g)
//   sum_t p_t v_t = sum_t (p_t s_tg) c_t + sum_t p_t m_tg
// so the matrix instructions work on the codes themselves, whole numbers 0..15
// that fp16 holds exactly, and s and m touch only the scores and the weights. A
// 4-bit code in the low mantissa bits of an fp16 is the (subnormal) number
// code * 2^-24, and four bits further up code * 2^-20: unpacking eight codes is
// one shift and four masks, and the powers of two go into the operands.
//
// The tokens (for the scores) and the channels (for the output) are the 16 rows of
// an m16n8k16, the 8 (query, head of the group) pairs of a CTA its columns. The
// weights come out with a token a row and go in with a token a column:
// movmatrix transposes them as fp16. fp32 outputs take q and p * s as hi + lo (22
// bits), fp16 ones p * s; bf16 outputs round at 2^-9 and do with the product of
// the fp16 weight and s.
//
// With codes 0..15 the two sums of an output are each about 4 sqrt(keys) times
// as large as what is left of them, and the matrix unit's 32-bit sums truncate
// (2.6e-5 of the result at 4097 keys): fp32 outputs take codes - 8 as values, and
// m + 8 s in 32-bit fmas.
//
// Each warp has a ring of its own of 32-token tiles, filled by untiled bulk
// copies: a block of 16 tokens of one head is contiguous, so the page table costs
// one look-up per 20 * d bytes and the loads no registers.
//
// The running maximum passes over a NaN score; the weights and their sum do not.
// A part (a warp's keys, a chunk's) whose sum is NaN joins the others with the
// reference +infinity, which makes its row NaN; -infinity is left to parts that
// saw no key.
#include "serve_ops.h"
#include "launch.cuh"
#include "serve_math.cuh"
#include "sm100.cuh"

#include <algorithm>
#include <atomic>
#include <climits>
#include <type_traits>

namespace vsb {

namespace {

constexpr int kKaWarps = 4, kKaThreads = 32 * kKaWarps;
constexpr int kKaTile = 32, kKaBlocks = kKaTile / kKv4Block;   // tokens a warp takes at a time
constexpr int kKaStages = 3;

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_f16_k8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(b0));
}

__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_h2(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }

// (a, b) as fp16 pairs hi + lo
__device__ __forceinline__ void split_h2(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = pack_h2(a, b);
    const float2 h = unpack_h2(hi);
    lo = pack_h2(a - h.x, b - h.y);
}

template <int N>
__device__ __forceinline__ void load_words(const void* p, uint32_t (&w)[N]) {
    static_assert(N == 2 || N == 4 || N == 8, "");
    if constexpr (N == 2) {
        const uint2 v = *static_cast<const uint2*>(p);
        w[0] = v.x; w[1] = v.y;
    } else {
        #pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const uint4 v = static_cast<const uint4*>(p)[i];
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
    }
}

// the same with the accumulator starting from zero
__device__ __forceinline__ void mma_f16_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_f16_k8_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(b0), "f"(0.f));
}

// 8 x 8 transpose of 16-bit elements: lane 4 r + c holds row r, columns 2 c and 2 c + 1
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// untiled bulk copy global -> shared (16-byte aligned, a multiple of 16 bytes)
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 :: "r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}

struct Kv4AttDev {
    Kv4AttArgs a;
    int group, rows, row_tiles, chunk, n_chunks;
    float2* part_ml;   // [batch][rows of all heads][n_chunks]: reference exponent and sum
    float* part_o;     // [batch][rows of all heads][n_chunks][d]
};

// this CTA's row -> query and head; how many keys it sees
__device__ __forceinline__ int row_limit(const Kv4AttArgs& a, int len, int query) {
    return a.causal ? min(max(len - a.queries + 1 + query, 0), len) : len;
}

// two codes (bits 0..3 and 16..19) minus 8 as fp16: 1024 + code is a whole fp16
__device__ __forceinline__ uint32_t centered_lo(uint32_t x) {
    const uint32_t v = (x & 0x000F000Fu) | 0x64006400u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v), __floats2half2_rn(1032.f, 1032.f));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// the same of bits 4..7 and 20..23: 1024 + 16 code
__device__ __forceinline__ uint32_t centered_hi(uint32_t x) {
    const uint32_t v = (x & 0x00F000F0u) | 0x64006400u;
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&v), __floats2half2_rn(0.0625f, 0.0625f),
                              __floats2half2_rn(-72.f, -72.f));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// what a warp has of its 8 rows at the end
template <int NG>
struct Kv4Joined {
    float o[8][NG * kKv4Group + 4], min[8][NG], sum[8], ref[8];
};

template <int NG>
__host__ __device__ constexpr int ka_smem() {   // the rings; the joined rows take their place at the end
    const int ring = kKaWarps * kKaStages * (kKaTile / kKv4Block) * 20 * NG * kKv4Group;
    const int red = kKaWarps * (int)sizeof(Kv4Joined<NG>);
    return ring > red ? ring : red;
}

// three CTAs an SM (168 registers) for 16-bit queries, two for fp32's two halves
template <int NG, typename T>
__global__ void __launch_bounds__(kKaThreads, std::is_same<T, float>::value ? 2 : 3)
kv4_attention_kernel(const __grid_constant__ Kv4AttDev p) {
    constexpr bool kF32Out = std::is_same<T, float>::value;
    constexpr bool kSplit = !std::is_same<T, __nv_bfloat16>::value;
    constexpr int D = NG * kKv4Group;
    constexpr int kBlockBytes = 20 * D, kTileBytes = kKaBlocks * kBlockBytes;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t bars[kKaWarps][kKaStages];
    const Kv4AttArgs& a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n = lane >> 2, quad = lane & 3;
    const int kvh = blockIdx.y / p.row_tiles, rt = blockIdx.y - kvh * p.row_tiles, b = blockIdx.z;
    if (lane < kKaStages) mbar_init(&bars[warp][lane], 1);
    fence_mbar_init();
    __syncwarp();
    pdl_trigger();
    pdl_wait();
    const int len = min(max(a.lens[b], 0), (int)min((long long)a.max_pages * a.cache.page, (long long)INT_MAX));
    // rows of this tile are (query, head) pairs in query order: the last one sees the most keys
    const int last_row = min(rt * 8 + 7, p.rows - 1);
    const int lim_max = row_limit(a, len, last_row / p.group);
    const int lim_min = row_limit(a, len, (rt * 8) / p.group);
    const int lo = blockIdx.x * p.chunk, hi = min(lo + p.chunk, lim_max);
    if (blockIdx.x > 0 && lo >= lim_max) return;

    // ---- the ring: lane i < kKaBlocks copies block i of a tile
    uint8_t* ring = smem + warp * (kKaStages * kTileBytes);
    const int* table = a.table + (long long)b * a.table_ld;
    const int page_shift = 31 - __clz(a.cache.page);
    auto look_up = [&](int t0) {   // the page of this lane's block, -1 past the end
        const int tb = t0 + lane * kKv4Block;
        return lane < kKaBlocks && tb < hi ? table[tb >> page_shift] : -1;
    };
    uint32_t there = 0;            // 4 bits a stage: the blocks that were copied
    auto fill = [&](int t0, int st, int pg) {
        const int tb = t0 + lane * kKv4Block;
        const bool want = lane < kKaBlocks && tb < hi;
        const bool in = want && (unsigned)pg < (unsigned long long)a.cache.n_pages;
        if (want && !in) record_status(kStatusBadShape);
        const uint32_t mask = __ballot_sync(0xffffffffu, in);
        if (lane == 0) mbar_arrive_expect_tx(&bars[warp][st], (uint32_t)(__popc(mask) * kBlockBytes));
        __syncwarp();
        if (in)
            bulk_load(ring + st * kTileBytes + lane * kBlockBytes,
                      a.cache.p + ((((long long)pg * a.cache.n_kv + kvh) << (page_shift - 4)) +
                                   ((tb & (a.cache.page - 1)) >> 4)) * kBlockBytes,
                      kBlockBytes, &bars[warp][st]);
        there = (there & ~(15u << (4 * st))) | mask << (4 * st);
    };
    constexpr int kStep = kKaWarps * kKaTile;
    const int first = lo + warp * kKaTile;
    int next = first;              // the tile to be copied next, and its pages
    int next_pg = look_up(next);
    #pragma unroll
    for (int st = 0; st < kKaStages; ++st)
        if (next < hi) {
            const int pg = next_pg, at = next;
            next += kStep;
            next_pg = look_up(next);
            fill(at, st, pg);
        }

    // column n: this lane's query row where it is an operand; rows 2 quad and
    // 2 quad + 1: the ones whose scores, sums and outputs it holds
    const int row = rt * 8 + n, query = row / p.group, head = kvh * p.group + row % p.group;
    const bool live = row < p.rows;
    const int lim = live ? row_limit(a, len, query) : 0;
    const int lim0 = __shfl_sync(0xffffffffu, lim, 8 * quad), lim1 = __shfl_sync(0xffffffffu, lim, 8 * quad + 4);

    // q of row n, channels 32 g + 8 quad + i: scaled by a power of two so that
    // the row's largest value lies in [2^9, 2^10) (sums of 32 stay in fp16). fp16
    // holds a scaled bf16 or fp16 value (down to 2^-24: 2^-33 of the largest).
    uint32_t qh[NG][4], ql[NG][4], qs = 0;
    float mul0, mul1;
    {
        float q[NG][8];
        float amax = 0.f;
        const T* src = static_cast<const T*>(a.q) + (long long)b * a.q_seq + (long long)query * a.q_tok +
                       (long long)head * a.q_head + 8 * quad;
        #pragma unroll
        for (int g = 0; g < NG; ++g)
            #pragma unroll
            for (int i = 0; i < 8; ++i) {
                q[g][i] = live ? to_f(src[32 * g + i]) : 0.f;
                amax = fmaxf(amax, fabsf(q[g][i]));
            }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // every finite query (the powers below stay normal numbers, a subnormal one keeps its bits)
        const int e = amax > 0.f ? min(max((int)(__float_as_uint(amax) >> 23) - 127, -117), 127) : 0;
        const float up = __uint_as_float((uint32_t)(127 + 9 - e) << 23);
        const float mul = a.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 - 9 + e) << 23);
        mul0 = __shfl_sync(0xffffffffu, mul, 8 * quad);
        mul1 = __shfl_sync(0xffffffffu, mul, 8 * quad + 4);
        float sums[NG];
        #pragma unroll
        for (int g = 0; g < NG; ++g) {
            sums[g] = 0.f;
            #pragma unroll
            for (int i = 0; i < 8; ++i) {
                q[g][i] *= up;
                sums[g] += q[g][i];
            }
            sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 1);
            sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 2);
            // nibbles (0, 4), (1, 5), (2, 6), (3, 7) come out of a word together;
            // those of odd index 16 times too large
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float f = (i & 1) ? 0.0625f : 1.0f;
                split_h2(q[g][i] * f, q[g][i + 4] * f, qh[g][i], ql[g][i]);
            }
        }
        // the K = 8 operand that meets the minima: the sums' hi parts on NG slots, their lo parts on the next NG
        #pragma unroll
        for (int g = 0; g < NG; g += 2) {
            uint32_t h, l;
            split_h2(sums[g], sums[g + 1], h, l);
            if (quad == g / 2) qs = h;
            if (quad == NG / 2 + g / 2) qs = l;
        }
    }

    float o[NG][2][4] = {};    // channels 32 g + 4 n + 2 h (+ 1) of rows 2 quad (+ 1)
    float mc[4] = {};          // sum p m of group n, and (n = 0) sum p, of rows 2 quad (+ 1)
    float vmin[NG] = {};       // the same of row n, tokens 2 quad (+ 1), where a product cannot give them:
    float l = 0.f;             // in tiles where a row ends (0 * NaN), and for fp32
    float m0 = -INFINITY, m1 = -INFINITY, ref0 = 0.f, ref1 = 0.f;
    // weights carry 2^ef, as large as weight <= 2^15 and weight * scale < 2^15 allow
    int ef = 15;
    bool ok = true;

    auto tile = [&](auto edge_tag, const uint8_t* tb, int t0, uint32_t in) {
        constexpr bool EDGE = decltype(edge_tag)::value;
        // ---- scores of 32 tokens: token 16 i + 8 j + n, rows 2 quad and 2 quad + 1
        float2 s[kKaBlocks][2];
        #pragma unroll
        for (int i = 0; i < kKaBlocks; ++i) {
            const uint8_t* blk = tb + i * kBlockBytes;
            uint32_t sc[2 * NG], w[2][NG];
            load_words(blk + 8 * D + (n >> 1) * (NG * 8), sc);
            load_words(blk + lane * (NG * 4), w[0]);
            load_words(blk + (32 + lane) * (NG * 4), w[1]);
            float mn[4];
            const uint32_t* km = reinterpret_cast<const uint32_t*>(blk + 9 * D) + n * NG + (quad & (NG / 2 - 1));
            mma_f16_k8_zero(mn, km[0], km[NG / 2], qs);
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
            #pragma unroll
            for (int g = 0; g < NG; ++g) {
                float acc[4];
                const uint32_t x0 = w[0][g], y0 = x0 >> 8, x1 = w[1][g], y1 = x1 >> 8;
                const uint32_t a0 = x0 & 0x000F000Fu, a1 = x1 & 0x000F000Fu, a2 = x0 & 0x00F000F0u, a3 = x1 & 0x00F000F0u;
                const uint32_t b0 = y0 & 0x000F000Fu, b1 = y1 & 0x000F000Fu, b2 = y0 & 0x00F000F0u, b3 = y1 & 0x00F000F0u;
                mma_f16_zero(acc, a0, a1, a2, a3, qh[g][0], qh[g][1]);
                mma_f16(acc, b0, b1, b2, b3, qh[g][2], qh[g][3]);
                if constexpr (kF32Out) {
                    mma_f16(acc, a0, a1, a2, a3, ql[g][0], ql[g][1]);
                    mma_f16(acc, b0, b1, b2, b3, ql[g][2], ql[g][3]);
                }
                // scales of tokens n and n + 8
                const float2 sg = unpack_h2(__byte_perm(sc[2 * g], sc[2 * g + 1], (n & 1) ? 0x7632u : 0x5410u));
                sum[0] = fmaf(sg.x, acc[0], sum[0]);
                sum[1] = fmaf(sg.x, acc[1], sum[1]);
                sum[2] = fmaf(sg.y, acc[2], sum[2]);
                sum[3] = fmaf(sg.y, acc[3], sum[3]);
            }
            #pragma unroll
            for (int j = 0; j < 2; ++j) {
                s[i][j].x = fmaf(sum[2 * j], 16777216.0f, mn[2 * j]) * mul0;
                s[i][j].y = fmaf(sum[2 * j + 1], 16777216.0f, mn[2 * j + 1]) * mul1;
                if constexpr (EDGE) {
                    const int t = t0 + i * kKv4Block + 8 * j + n;
                    if (t >= lim0 || !(in >> i & 1u)) s[i][j].x = -INFINITY;
                    if (t >= lim1 || !(in >> i & 1u)) s[i][j].y = -INFINITY;
                }
            }
        }
        // ---- weights 2^(s - max + ef)
        float mt0 = m0, mt1 = m1;
        __half2 top = __floats2half2_rn(0.f, 0.f);
        #pragma unroll
        for (int i = 0; i < kKaBlocks; ++i) {
            mt0 = fmaxf(mt0, fmaxf(s[i][0].x, s[i][1].x));
            mt1 = fmaxf(mt1, fmaxf(s[i][0].y, s[i][1].y));
            // the largest scale of the tile: each lane one word (a scale that is NaN counts as 0)
            uint32_t x = *reinterpret_cast<const uint32_t*>(tb + i * kBlockBytes + 18 * D + quad * (NG * 8) +
                                                           (n & (2 * NG - 1)) * 4);
            if constexpr (EDGE) {   // past the end the bytes are anything
                const int t = t0 + i * kKv4Block + 8 * (n & 1) + 2 * quad;
                if (t >= len || !(in >> i & 1u)) x = 0u;
                else if (t + 1 >= len) x &= 0xFFFFu;
            }
            top = __hmax2(top, *reinterpret_cast<const __half2*>(&x));
        }
        #pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
            mt0 = fmaxf(mt0, __shfl_xor_sync(0xffffffffu, mt0, x));
            mt1 = fmaxf(mt1, __shfl_xor_sync(0xffffffffu, mt1, x));
        }
        const __half top1 = __hmax(__low2half(top), __high2half(top));
        const uint32_t smax = __reduce_max_sync(0xffffffffu, (uint32_t)__half_as_ushort(top1));   // positive: bits order
        if (smax >= 0x0400u && smax < 0x7C00u) ef = min(ef, 14 - ((int)(smax >> 10) - 15));
        const float new0 = mt0 == -INFINITY ? 0.f : mt0 - (float)ef, new1 = mt1 == -INFINITY ? 0.f : mt1 - (float)ef;
        if (__any_sync(0xffffffffu, new0 != ref0 || new1 != ref1)) {
            const float al0 = m0 == -INFINITY ? 0.f : ex2(ref0 - new0), al1 = m1 == -INFINITY ? 0.f : ex2(ref1 - new1);
            #pragma unroll
            for (int e = 0; e < 4; ++e) {
                mc[e] *= (e & 1) ? al1 : al0;
                #pragma unroll
                for (int g = 0; g < NG; ++g) {
                    o[g][0][e] *= (e & 1) ? al1 : al0;
                    o[g][1][e] *= (e & 1) ? al1 : al0;
                }
            }
            const float x0 = __shfl_sync(0xffffffffu, al0, n >> 1), x1 = __shfl_sync(0xffffffffu, al1, n >> 1);
            const float aln = (n & 1) ? x1 : x0;
            l *= aln;
            #pragma unroll
            for (int g = 0; g < NG; ++g) vmin[g] *= aln;
        }
        m0 = mt0;
        m1 = mt1;
        ref0 = new0;
        ref1 = new1;
        // ---- weights times codes
        #pragma unroll
        for (int i = 0; i < kKaBlocks; ++i) {
            const uint8_t* blk = tb + i * kBlockBytes;
            if (EDGE && !(in >> i & 1u)) continue;
            uint32_t ph[2], pl[2];   // fp16 weights of row n, tokens 8 j + 2 quad (+ 1), and what they leave
            #pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float x = ex2(s[i][j].x - ref0), y = ex2(s[i][j].y - ref1);
                split_h2(x, y, ph[j], pl[j]);
                ph[j] = transpose_8x8(ph[j]);
                if constexpr (kSplit) pl[j] = transpose_8x8(pl[j]);
            }
            uint32_t vs[2 * NG], w[2][NG];
            load_words(blk + 18 * D + quad * (NG * 8), vs);
            load_words(blk + 10 * D + lane * (NG * 4), w[0]);
            load_words(blk + 10 * D + (32 + lane) * (NG * 4), w[1]);
            if constexpr (EDGE) {   // a token that a row does not see adds nothing to it, whatever its scale is
                const int t = t0 + i * kKv4Block + 2 * quad;
                const uint32_t k0 = (t < lim ? 0xFFFFu : 0u) | (t + 1 < lim ? 0xFFFF0000u : 0u);
                const uint32_t k1 = (t + 8 < lim ? 0xFFFFu : 0u) | (t + 9 < lim ? 0xFFFF0000u : 0u);
                #pragma unroll
                for (int g = 0; g < NG; ++g) {
                    vs[2 * g] &= k0;
                    vs[2 * g + 1] &= k1;
                }
            }
            float2 pw[2];
            #pragma unroll
            for (int j = 0; j < 2; ++j) {
                pw[j] = unpack_h2(ph[j]);
                if constexpr (kSplit) {
                    const float2 x = unpack_h2(pl[j]);
                    pw[j].x += x.x;
                    pw[j].y += x.y;
                }
            }
            if constexpr (EDGE || kF32Out) {
                const int t = t0 + i * kKv4Block + 2 * quad;
                uint32_t vm[2 * NG];
                load_words(blk + 19 * D + quad * (NG * 8), vm);
                #pragma unroll
                for (int j = 0; j < 2; ++j) {
                    l += pw[j].x + pw[j].y;
                    #pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        float2 mm = unpack_h2(vm[2 * g + j]);
                        if constexpr (kF32Out) mm = fma2(unpack_h2(vs[2 * g + j]), make_float2(8.f, 8.f), mm);
                        if constexpr (EDGE) {
                            if (t + 8 * j >= lim) mm.x = 0.f;
                            if (t + 8 * j + 1 >= lim) mm.y = 0.f;
                        }
                        vmin[g] = fmaf(pw[j].x, mm.x, fmaf(pw[j].y, mm.y, vmin[g]));
                    }
                }
            } else {
                // minima of group n (token pairs are words already); ones in row 8 for the sum
                uint2 am = make_uint2(0u, 0u);
                if (n < NG) am = *reinterpret_cast<const uint2*>(blk + 19 * D + (quad * NG + n) * 8);
                const uint32_t one = n == 0 ? 0x3C003C00u : 0u;
                mma_f16(mc, am.x, one, am.y, one, ph[0], ph[1]);
                if constexpr (kSplit) mma_f16(mc, am.x, one, am.y, one, pl[0], pl[1]);
            }
            #pragma unroll
            for (int g = 0; g < NG; ++g) {
                uint32_t b0, b1;                          // p * s of row n
                [[maybe_unused]] uint32_t c0 = 0u, c1 = 0u;   // and what it leaves
                if constexpr (kSplit) {
                    const float2 s0 = unpack_h2(vs[2 * g]), s1 = unpack_h2(vs[2 * g + 1]);
                    split_h2(pw[0].x * s0.x, pw[0].y * s0.y, b0, c0);
                    split_h2(pw[1].x * s1.x, pw[1].y * s1.y, b1, c1);
                } else {
                    b0 = mul_h2(ph[0], vs[2 * g]);
                    b1 = mul_h2(ph[1], vs[2 * g + 1]);
                }
                const uint32_t x0 = w[0][g], y0 = x0 >> 8, x1 = w[1][g], y1 = x1 >> 8;
                uint32_t c[8];
                if constexpr (kF32Out) {
                    c[0] = centered_lo(x0); c[1] = centered_hi(x0); c[2] = centered_lo(x1); c[3] = centered_hi(x1);
                    c[4] = centered_lo(y0); c[5] = centered_hi(y0); c[6] = centered_lo(y1); c[7] = centered_hi(y1);
                } else {
                    c[0] = x0 & 0x000F000Fu; c[1] = x0 & 0x00F000F0u; c[2] = x1 & 0x000F000Fu; c[3] = x1 & 0x00F000F0u;
                    c[4] = y0 & 0x000F000Fu; c[5] = y0 & 0x00F000F0u; c[6] = y1 & 0x000F000Fu; c[7] = y1 & 0x00F000F0u;
                }
                mma_f16(o[g][0], c[0], c[1], c[2], c[3], b0, b1);
                mma_f16(o[g][1], c[4], c[5], c[6], c[7], b0, b1);
                if constexpr (kSplit) {
                    mma_f16(o[g][0], c[0], c[1], c[2], c[3], c0, c1);
                    mma_f16(o[g][1], c[4], c[5], c[6], c[7], c0, c1);
                }
            }
        }
    };

    int st = 0;
    uint32_t phase = 0;
    for (int t0 = first; t0 < hi; t0 += kStep) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bars[warp][st], phase)) != 0;
        if (!ok) break;
        const uint32_t in = there >> (4 * st) & 15u;
        const uint8_t* tb = ring + st * kTileBytes;
        if (t0 + kKaTile <= lim_min && in == (1u << kKaBlocks) - 1u)
            tile(std::false_type{}, tb, t0, in);
        else
            tile(std::true_type{}, tb, t0, in);
        __syncwarp();   // the stage is free
        if (next < hi) {
            const int pg = next_pg, at = next;
            next += kStep;
            next_pg = look_up(next);
            fill(at, st, pg);
        }
        if (++st == kKaStages) {
            st = 0;
            phase ^= 1;
        }
    }
    if (!ok) {   // after a wait that gave up: the copies still have to land
        const uint64_t until = globaltimer_ns() + kWaitLimitNs;
        for (int x = 0; x < kKaStages; ++x) {
            mbar_wait_until(&bars[warp][x], 0, until);
            mbar_wait_until(&bars[warp][x], 1, until);
        }
    }

    // ---- join the warps: every row's parts on the largest reference
    __syncthreads();
    Kv4Joined<NG>* red = reinterpret_cast<Kv4Joined<NG>*>(smem);
    Kv4Joined<NG>& mine = red[warp];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    #pragma unroll
    for (int g = 0; g < NG; ++g) {
        vmin[g] += __shfl_xor_sync(0xffffffffu, vmin[g], 1);
        vmin[g] += __shfl_xor_sync(0xffffffffu, vmin[g], 2);
        if (quad == 0) mine.min[n][g] = vmin[g];
    }
    if (quad == 0) mine.sum[n] = l;
    __syncwarp();
    if (n < NG) {
        mine.min[2 * quad][n] += mc[0];
        mine.min[2 * quad + 1][n] += mc[1];
    }
    if (n == 0) {
        const float sum0 = mine.sum[2 * quad] + mc[2], sum1 = mine.sum[2 * quad + 1] + mc[3];
        mine.sum[2 * quad] = sum0;
        mine.sum[2 * quad + 1] = sum1;
        mine.ref[2 * quad] = sum0 != sum0 ? INFINITY : m0 == -INFINITY ? -INFINITY : ref0;
        mine.ref[2 * quad + 1] = sum1 != sum1 ? INFINITY : m1 == -INFINITY ? -INFINITY : ref1;
    }
    __syncwarp();
    #pragma unroll
    for (int g = 0; g < NG; ++g)
        #pragma unroll
        for (int h = 0; h < 2; ++h)
            #pragma unroll
            for (int e = 0; e < 4; ++e) {   // channels of odd index came 16 times too large
                const int r = 2 * quad + (e & 1);
                const float f = kF32Out ? 1.0f : (e >> 1) ? 1048576.0f : 16777216.0f;
                mine.o[r][32 * g + 4 * n + 2 * h + (e >> 1)] = fmaf(o[g][h][e], f, mine.min[r][g]);
            }
    __syncthreads();
    constexpr int kLanes = kKaThreads / 8;   // threads of one row
    const int r = tid / kLanes, rl = tid % kLanes, rrow = rt * 8 + r;
    if (rrow >= p.rows) return;
    float rmax = -INFINITY;
    #pragma unroll
    for (int w = 0; w < kKaWarps; ++w) rmax = fmaxf(rmax, red[w].ref[r]);
    float wt[kKaWarps], lsum = 0.f;
    #pragma unroll
    for (int w = 0; w < kKaWarps; ++w) {   // a warp that saw no key: the weight -1, left out
        wt[w] = red[w].ref[r] == -INFINITY ? -1.f : ex2(red[w].ref[r] - rmax);
        lsum = wt[w] < 0.f ? lsum : fmaf(red[w].sum[r], wt[w], lsum);
    }
    const int rq = rrow / p.group, rh = kvh * p.group + rrow % p.group;
    const long long out_row = ((long long)b * a.queries + rq) * a.n_q + rh;
    const bool direct = p.n_chunks == 1;
    const float inv = !direct ? 1.f : rmax == -INFINITY ? 0.f : 1.0f / lsum;
    T* out = static_cast<T*>(a.out) + out_row * D;
    float* part = p.part_o + (out_row * p.n_chunks + blockIdx.x) * D;
    for (int c = rl; c < D; c += kLanes) {
        float v = 0.f;
        #pragma unroll
        for (int w = 0; w < kKaWarps; ++w) v = wt[w] < 0.f ? v : fmaf(red[w].o[r][c], wt[w], v);
        if (direct) out[c] = from_f<T>(v * inv);
        else part[c] = v;
    }
    if (!direct && rl == 0) p.part_ml[out_row * p.n_chunks + blockIdx.x] = make_float2(rmax, lsum);
}

// Joins the chunks of a row, in order: one warp a row.
template <int NG, typename T>
__global__ void __launch_bounds__(128)
kv4_attention_join_kernel(const __grid_constant__ Kv4AttDev p) {
    constexpr int D = NG * kKv4Group;
    const Kv4AttArgs& a = p.a;
    const int lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    pdl_trigger();
    pdl_wait();
    if (row >= (long long)a.batch * a.queries * a.n_q) return;
    const int query = (int)(row / a.n_q % a.queries), b = (int)(row / a.n_q / a.queries);
    const int len = min(max(a.lens[b], 0), (int)min((long long)a.max_pages * a.cache.page, (long long)INT_MAX));
    const int n = min((row_limit(a, len, query) + p.chunk - 1) / p.chunk, p.n_chunks);
    float ref = -INFINITY;
    for (int c = lane; c < n; c += 32) ref = fmaxf(ref, p.part_ml[row * p.n_chunks + c].x);
    for (int x = 16; x > 0; x >>= 1) ref = fmaxf(ref, __shfl_xor_sync(0xffffffffu, ref, x));
    float v[NG] = {}, l = 0.f;
    for (int c = 0; c < n; ++c) {
        const float2 ml = p.part_ml[row * p.n_chunks + c];
        if (ml.x == -INFINITY) continue;
        const float w = ex2(ml.x - ref);
        l = fmaf(ml.y, w, l);
        const float* part = p.part_o + (row * p.n_chunks + c) * D;
        #pragma unroll
        for (int g = 0; g < NG; ++g) v[g] = fmaf(part[32 * g + lane], w, v[g]);
    }
    const float inv = ref == -INFINITY ? 0.f : 1.0f / l;
    #pragma unroll
    for (int g = 0; g < NG; ++g) static_cast<T*>(a.out)[row * D + 32 * g + lane] = from_f<T>(v[g] * inv);
}

template <int NG, typename T>
cudaError_t kv4_launch(const Kv4AttDev& p, dim3 grid, cudaStream_t st) {
    static std::atomic<unsigned long long> ready{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(ready.load() & bit)) {
        e = cudaFuncSetAttribute(kv4_attention_kernel<NG, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, ka_smem<NG>());
        if (e != cudaSuccess) return e;
        ready.fetch_or(bit);
    }
    return launch_k(kv4_attention_kernel<NG, T>, grid, dim3(kKaThreads), ka_smem<NG>(), st, p);
}

// Keys a CTA takes, from the width of the table (the lengths are on the device).
// Chunks down to a tile of each warp fill one wave of three CTAs an SM (fp32
// queries have two: theirs is a wave and a half). Latency: one sequence of 1021
// tokens, 5 heads: 6.9 us in 8 chunks, 7.2 in 4, 10.3 whole. Beyond a wave chunks
// only even out the tail, which pays while they stay near 1000 keys (16
// sequences of up to 8192, 8 heads: 24.3 us in 8 chunks of 1024; 896: 25.5,
// 1664: 29.6, 512: 28.5, whole: 66) and not at 128 (8 sequences of 256 with 19 row
// tiles: 12.3 us whole, 21.2 in chunks of 128).
int kv4_chunk(int batch, int row_ctas, long long max_len) {
    const long long tile = (long long)kKaTile * kKaWarps, ctas = (long long)batch * row_ctas;
    const long long fill = std::min((148 * 3 + ctas - 1) / ctas, max_len / tile);
    const long long even = std::min((148 * 8 + ctas - 1) / ctas, max_len / 896);
    const long long want = std::max({fill, even, 1ll});
    const long long chunk = (max_len + want - 1) / want;
    return (int)std::max((chunk + tile - 1) / tile * tile, tile);
}

}  // namespace

unsigned long long kv4_attention_ws_bytes(int batch, int queries, int n_q, int n_kv, int d, long long max_len) {
    if (batch <= 0 || queries <= 0 || max_len <= 0) return 0;
    const int row_tiles = (queries * (n_q / n_kv) + 7) / 8;
    const int chunk = kv4_chunk(batch, n_kv * row_tiles, max_len);
    const unsigned long long n_chunks = (unsigned long long)((max_len + chunk - 1) / chunk);
    return n_chunks == 1 ? 0 : (unsigned long long)batch * queries * n_q * n_chunks * (d + 2) * sizeof(float);
}

cudaError_t kv4_attention(const Kv4AttArgs& a, cudaStream_t st) {
    if (a.batch <= 0 || a.queries <= 0) return cudaSuccess;
    Kv4AttDev p;
    p.a = a;
    p.group = a.n_q / a.cache.n_kv;
    p.rows = a.queries * p.group;
    p.row_tiles = (p.rows + 7) / 8;
    const long long max_len = (long long)a.max_pages * a.cache.page;
    p.chunk = kv4_chunk(a.batch, a.cache.n_kv * p.row_tiles, max_len);
    p.n_chunks = max_len > 0 ? (int)((max_len + p.chunk - 1) / p.chunk) : 1;
    const long long rows = (long long)a.batch * a.queries * a.n_q;
    p.part_ml = static_cast<float2*>(a.ws);
    p.part_o = reinterpret_cast<float*>(p.part_ml + rows * p.n_chunks);
    if (p.n_chunks > 1 &&
        (!a.ws || a.ws_bytes < (unsigned long long)rows * p.n_chunks * (a.cache.d + 2) * sizeof(float)))
        return cudaErrorInvalidValue;
    const dim3 grid((unsigned)p.n_chunks, (unsigned)(a.cache.n_kv * p.row_tiles), (unsigned)a.batch);
    const cudaError_t e = by_type(a.type, [&](auto t) {
        using T = decltype(t);
        cudaError_t r = a.cache.d == 128 ? kv4_launch<4, T>(p, grid, st) : kv4_launch<2, T>(p, grid, st);
        if (r != cudaSuccess || p.n_chunks == 1) return r;
        const dim3 jgrid((unsigned)((rows + 3) / 4));
        return a.cache.d == 128 ? launch_k(kv4_attention_join_kernel<4, T>, jgrid, dim3(128), 0, st, p)
                                : launch_k(kv4_attention_join_kernel<2, T>, jgrid, dim3(128), 0, st, p);
    });
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace vsb

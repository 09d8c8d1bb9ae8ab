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
// Rows are 8 (query, head of the group) pairs. m16n8k16 has 16: the other 8
// carry what the fp16 rounding of the first 8 left (q and p * s as hi + lo, 22
// bits), so scores and weights are 32-bit quality at no further instruction.
//
// With codes 0..15 the two sums of an output are each about 4 sqrt(keys) times
// as large as what is left of them, and the matrix unit's 32-bit sums truncate:
// 2.6e-5 of the result at 4097 keys. fp16 and bf16 outputs do not see that;
// fp32 ones take codes - 8 as values (and m + 8 s), one more instruction for
// every two codes.
#include "serve_ops.h"
#include "launch.cuh"
#include "sm100.cuh"

#include <climits>
#include <type_traits>

namespace vsb {

namespace {

constexpr int kKaWarps = 4, kKaThreads = 32 * kKaWarps;
constexpr int kKaTile = 64, kKaBlocks = kKaTile / kKv4Block;   // tokens a warp takes at a time

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

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

template <int NG, typename T, bool SPLIT, bool CENTER>
__global__ void __launch_bounds__(kKaThreads)
kv4_attention_kernel(const __grid_constant__ Kv4AttDev p) {
    constexpr int D = NG * kKv4Group;
    constexpr int kBlockBytes = 20 * D;
    __shared__ float red[kKaWarps][8][D + 2];
    const Kv4AttArgs& a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n = lane >> 2, quad = lane & 3;
    const int kvh = blockIdx.y / p.row_tiles, rt = blockIdx.y - kvh * p.row_tiles, b = blockIdx.z;
    pdl_trigger();
    pdl_wait();
    const int len = min(max(a.lens[b], 0), (int)min((long long)a.max_pages * a.cache.page, (long long)INT_MAX));
    // rows of this tile are (query, head) pairs in query order: the last one sees the most keys
    const int last_row = min(rt * 8 + 7, p.rows - 1);
    const int lim_max = row_limit(a, len, last_row / p.group);
    const int lo = blockIdx.x * p.chunk, hi = min(lo + p.chunk, lim_max);
    if (blockIdx.x > 0 && lo >= lim_max) return;

    const int row = rt * 8 + n, query = row / p.group, head = kvh * p.group + row % p.group;
    const bool live = row < p.rows;
    const int lim = live ? row_limit(a, len, query) : 0;

    // q of row n, channels 32 g + 8 quad + i: scaled by a power of two so that
    // the row's largest value lies in [2^9, 2^10) (sums of 32 stay in fp16)
    uint32_t qh[NG][4], ql[NG][4];
    uint32_t qsh = 0, qsl = 0;   // sums of the groups 2 quad, 2 quad + 1 (the K = 8 operand)
    float row_mul;
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
        const int e = amax > 0.f ? min(max((int)(__float_as_uint(amax) >> 23) - 127, -100), 100) : 0;
        const float up = __uint_as_float((uint32_t)(127 + 9 - e) << 23);
        row_mul = a.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 - 9 + e) << 23);
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
        #pragma unroll
        for (int g = 0; g < NG; g += 2)
            if (quad == g / 2) split_h2(sums[g], sums[g + 1], qsh, qsl);
    }

    float o[NG][4][4] = {};
    float vmin[NG] = {};
    float l = 0.f, m = -INFINITY, ref = 0.f;
    int ef = 40;   // weights carry 2^ef: weight * scale then fills fp16's range (see below)
    const int* table = a.table + (long long)b * a.table_ld;
    const int page_blocks = a.cache.page / kKv4Block;
    for (int t0 = lo + warp * kKaTile; t0 < hi; t0 += kKaWarps * kKaTile) {
        const bool edge = t0 + kKaTile > row_limit(a, len, (rt * 8) / p.group);   // some row may end in this tile
        const uint8_t* blk[kKaBlocks];
        #pragma unroll
        for (int i = 0; i < kKaBlocks; ++i) {
            const int tb = t0 + i * kKv4Block;
            blk[i] = nullptr;
            if (tb < hi) {
                const int pg = tb / a.cache.page;
                const int at = table[pg];
                if ((unsigned)at < (unsigned long long)a.cache.n_pages)
                    blk[i] = a.cache.p + (((long long)at * a.cache.n_kv + kvh) * page_blocks +
                                          (tb - pg * a.cache.page) / kKv4Block) * kBlockBytes;
                else
                    record_status(kStatusBadShape);
            }
        }
        // ---- scores of 64 tokens: this lane row n, tokens 16 i + 8 j + 2 quad + {0, 1}
        float s[kKaBlocks][2][2];
        #pragma unroll
        for (int i = 0; i < kKaBlocks; ++i) {
            #pragma unroll
            for (int j = 0; j < 2; ++j) s[i][j][0] = s[i][j][1] = -INFINITY;
            if (!blk[i]) continue;
            uint32_t sc[2 * NG];
            load_words(blk[i] + 8 * D + quad * (NG * 8), sc);
            #pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t w[NG];
                load_words(blk[i] + (j * 32 + lane) * (NG * 4), w);
                float mn[4] = {};
                const uint32_t bm = 2 * quad < NG
                    ? *reinterpret_cast<const uint32_t*>(blk[i] + 9 * D + ((n * 2 + j) * NG + 2 * quad) * 2) : 0u;
                mma_f16_k8(mn, qsh, qsl, bm);
                float t0s = 0.f, t1s = 0.f;
                #pragma unroll
                for (int g = 0; g < NG; ++g) {
                    float acc[4] = {};
                    const uint32_t x = w[g], y = w[g] >> 8;
                    mma_f16(acc, qh[g][0], ql[g][0], qh[g][1], ql[g][1], x & 0x000F000Fu, x & 0x00F000F0u);
                    mma_f16(acc, qh[g][2], ql[g][2], qh[g][3], ql[g][3], y & 0x000F000Fu, y & 0x00F000F0u);
                    const float2 sg = unpack_h2(sc[g * 2 + j]);
                    t0s = fmaf(sg.x, acc[0] + acc[2], t0s);
                    t1s = fmaf(sg.y, acc[1] + acc[3], t1s);
                }
                s[i][j][0] = fmaf(t0s, 16777216.0f, mn[0] + mn[2]) * row_mul;
                s[i][j][1] = fmaf(t1s, 16777216.0f, mn[1] + mn[3]) * row_mul;
                if (edge) {
                    const int t = t0 + i * kKv4Block + 8 * j + 2 * quad;
                    if (t >= lim) s[i][j][0] = -INFINITY;
                    if (t + 1 >= lim) s[i][j][1] = -INFINITY;
                }
            }
        }
        // ---- weights 2^(s - max) * 2^ef, ef as large as p * scale < 2^15 allows
        float mt = m;
        #pragma unroll
        for (int i = 0; i < kKaBlocks; ++i)
            #pragma unroll
            for (int j = 0; j < 2; ++j) mt = fmaxf(mt, fmaxf(s[i][j][0], s[i][j][1]));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
        uint32_t vs[kKaBlocks][2 * NG];
        __half2 top = __floats2half2_rn(0.f, 0.f);
        #pragma unroll
        for (int i = 0; i < kKaBlocks; ++i) {
            #pragma unroll
            for (int x = 0; x < 2 * NG; ++x) vs[i][x] = 0u;
            if (!blk[i]) continue;
            load_words(blk[i] + 18 * D + quad * (NG * 8), vs[i]);
            #pragma unroll
            for (int x = 0; x < 2 * NG; ++x) {
                if (edge) {   // past the end the bytes are anything
                    const int t = t0 + i * kKv4Block + 8 * (x & 1) + 2 * quad;
                    if (t >= len) vs[i][x] = 0u;
                    else if (t + 1 >= len) vs[i][x] &= 0xFFFFu;
                }
                top = __hmax2(top, *reinterpret_cast<const __half2*>(&vs[i][x]));
            }
        }
        float smax = fmaxf(__low2float(top), __high2float(top));
        smax = fmaxf(smax, __shfl_xor_sync(0xffffffffu, smax, 1));
        smax = fmaxf(smax, __shfl_xor_sync(0xffffffffu, smax, 2));
        if (smax > 0.f && smax < 131072.f) ef = min(ef, 14 - ((int)(__float_as_uint(smax) >> 23) - 127));
        const float ref_new = mt == -INFINITY ? 0.f : mt - (float)ef;
        if (__any_sync(0xffffffffu, ref_new != ref)) {
            const float alpha = m == -INFINITY ? 0.f : ex2(ref - ref_new);
            l *= alpha;
            #pragma unroll
            for (int g = 0; g < NG; ++g) {
                vmin[g] *= alpha;
                #pragma unroll
                for (int i = 0; i < 4; ++i)
                    #pragma unroll
                    for (int e = 0; e < 4; ++e) o[g][i][e] *= alpha;
            }
        }
        m = mt;
        ref = ref_new;
        // ---- weights times codes
        #pragma unroll
        for (int i = 0; i < kKaBlocks; ++i) {
            if (!blk[i]) continue;
            float pw[2][2];
            #pragma unroll
            for (int j = 0; j < 2; ++j)
                #pragma unroll
                for (int e = 0; e < 2; ++e) {
                    pw[j][e] = ex2(s[i][j][e] - ref);
                    l += pw[j][e];
                }
            uint32_t vm[2 * NG], w[2][NG];
            load_words(blk[i] + 19 * D + quad * (NG * 8), vm);
            load_words(blk[i] + 10 * D + lane * (NG * 4), w[0]);
            load_words(blk[i] + 10 * D + (32 + lane) * (NG * 4), w[1]);
            #pragma unroll
            for (int g = 0; g < NG; ++g) {
                float2 s0 = unpack_h2(vs[i][2 * g]), s1 = unpack_h2(vs[i][2 * g + 1]);
                float2 m0 = unpack_h2(vm[2 * g]), m1 = unpack_h2(vm[2 * g + 1]);
                if constexpr (CENTER) {
                    m0.x = fmaf(8.f, s0.x, m0.x);
                    m0.y = fmaf(8.f, s0.y, m0.y);
                    m1.x = fmaf(8.f, s1.x, m1.x);
                    m1.y = fmaf(8.f, s1.y, m1.y);
                }
                if (edge) {   // a token a row does not see adds nothing to it, whatever it holds
                    const int t = t0 + i * kKv4Block + 2 * quad;
                    if (t >= lim) s0.x = m0.x = 0.f;
                    if (t + 1 >= lim) s0.y = m0.y = 0.f;
                    if (t + 8 >= lim) s1.x = m1.x = 0.f;
                    if (t + 9 >= lim) s1.y = m1.y = 0.f;
                }
                vmin[g] = fmaf(pw[0][0], m0.x, fmaf(pw[0][1], m0.y, fmaf(pw[1][0], m1.x, fmaf(pw[1][1], m1.y, vmin[g]))));
                uint32_t a0, a1 = 0u, a2, a3 = 0u;
                if constexpr (SPLIT) {
                    split_h2(pw[0][0] * s0.x, pw[0][1] * s0.y, a0, a1);
                    split_h2(pw[1][0] * s1.x, pw[1][1] * s1.y, a2, a3);
                } else {
                    a0 = pack_h2(pw[0][0] * s0.x, pw[0][1] * s0.y);
                    a2 = pack_h2(pw[1][0] * s1.x, pw[1][1] * s1.y);
                }
                const uint32_t x0 = w[0][g], y0 = x0 >> 8, x1 = w[1][g], y1 = x1 >> 8;
                if constexpr (CENTER) {
                    mma_f16(o[g][0], a0, a1, a2, a3, centered_lo(x0), centered_lo(x1));
                    mma_f16(o[g][1], a0, a1, a2, a3, centered_hi(x0), centered_hi(x1));
                    mma_f16(o[g][2], a0, a1, a2, a3, centered_lo(y0), centered_lo(y1));
                    mma_f16(o[g][3], a0, a1, a2, a3, centered_hi(y0), centered_hi(y1));
                } else {
                    mma_f16(o[g][0], a0, a1, a2, a3, x0 & 0x000F000Fu, x1 & 0x000F000Fu);
                    mma_f16(o[g][1], a0, a1, a2, a3, x0 & 0x00F000F0u, x1 & 0x00F000F0u);
                    mma_f16(o[g][2], a0, a1, a2, a3, y0 & 0x000F000Fu, y1 & 0x000F000Fu);
                    mma_f16(o[g][3], a0, a1, a2, a3, y0 & 0x00F000F0u, y1 & 0x00F000F0u);
                }
            }
        }
    }

    // ---- join the warps: every row's parts on the largest reference
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    #pragma unroll
    for (int g = 0; g < NG; ++g) {
        vmin[g] += __shfl_xor_sync(0xffffffffu, vmin[g], 1);
        vmin[g] += __shfl_xor_sync(0xffffffffu, vmin[g], 2);
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float f = CENTER ? 1.0f : (i & 1) ? 1048576.0f : 16777216.0f;
            red[warp][n][32 * g + 8 * quad + i] = fmaf(o[g][i][0] + o[g][i][2], f, vmin[g]);
            red[warp][n][32 * g + 8 * quad + 4 + i] = fmaf(o[g][i][1] + o[g][i][3], f, vmin[g]);
        }
    }
    if (quad == 0) {
        red[warp][n][D] = m == -INFINITY ? -INFINITY : ref;
        red[warp][n][D + 1] = l;
    }
    __syncthreads();
    constexpr int kLanes = kKaThreads / 8;   // threads of one row
    const int r = tid / kLanes, rl = tid % kLanes, rrow = rt * 8 + r;
    if (rrow >= p.rows) return;
    float rmax = -INFINITY;
    #pragma unroll
    for (int w = 0; w < kKaWarps; ++w) rmax = fmaxf(rmax, red[w][r][D]);
    float wt[kKaWarps], lsum = 0.f;
    #pragma unroll
    for (int w = 0; w < kKaWarps; ++w) {
        wt[w] = red[w][r][D] == -INFINITY ? 0.f : ex2(red[w][r][D] - rmax);
        lsum = fmaf(red[w][r][D + 1], wt[w], lsum);
    }
    const int rq = rrow / p.group, rh = kvh * p.group + rrow % p.group;
    const long long out_row = ((long long)b * a.queries + rq) * a.n_q + rh;
    if (p.n_chunks == 1) {
        T* out = static_cast<T*>(a.out) + out_row * D;
        const float inv = rmax == -INFINITY ? 0.f : 1.0f / lsum;
        for (int c = rl; c < D; c += kLanes) {
            float v = 0.f;
            #pragma unroll
            for (int w = 0; w < kKaWarps; ++w) v = wt[w] == 0.f ? v : fmaf(red[w][r][c], wt[w], v);
            out[c] = from_f<T>(v * inv);
        }
    } else {
        float* part = p.part_o + (out_row * p.n_chunks + blockIdx.x) * D;
        for (int c = rl; c < D; c += kLanes) {
            float v = 0.f;
            #pragma unroll
            for (int w = 0; w < kKaWarps; ++w) v = wt[w] == 0.f ? v : fmaf(red[w][r][c], wt[w], v);
            part[c] = v;
        }
        if (rl == 0) p.part_ml[out_row * p.n_chunks + blockIdx.x] = make_float2(rmax, lsum);
    }
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

// Keys a CTA takes: as many chunks as fill the SMs about four times over, none
// shorter than one tile of each warp.
int kv4_chunk(int batch, int row_ctas, long long max_len) {
    const long long tile = (long long)kKaTile * kKaWarps;
    long long want = (148ll * 8 + (long long)batch * row_ctas - 1) / ((long long)batch * row_ctas);
    long long chunk = (max_len + want - 1) / want;
    chunk = (chunk + tile - 1) / tile * tile;
    return (int)(chunk < tile ? tile : chunk);
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
        // bf16 outputs round at 2^-9: the weights' fp16 rounding (2^-12) needs no second part
        constexpr bool split = !std::is_same<T, __nv_bfloat16>::value, center = std::is_same<T, float>::value;
        cudaError_t r = a.cache.d == 128
            ? launch_k(kv4_attention_kernel<4, T, split, center>, grid, dim3(kKaThreads), 0, st, p)
            : launch_k(kv4_attention_kernel<2, T, split, center>, grid, dim3(kKaThreads), 0, st, p);
        if (r != cudaSuccess || p.n_chunks == 1) return r;
        const dim3 jgrid((unsigned)((rows + 3) / 4));
        return a.cache.d == 128 ? launch_k(kv4_attention_join_kernel<4, T>, jgrid, dim3(128), 0, st, p)
                                : launch_k(kv4_attention_join_kernel<2, T>, jgrid, dim3(128), 0, st, p);
    });
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace vsb

// Head norms with multi-axis rotary positions, and the append / read operators
// of the paged 4-bit cache. All of them move each value once; what bounds them
// is HBM at prompt sizes and the launch at single tokens.
#include "serve_ops.h"
#include "launch.cuh"
#include "serve_math.cuh"
#include "sm100.cuh"

#include <algorithm>
#include <climits>
#include <cstdlib>

namespace vsb {

namespace {

// N consecutive elements as one access (p aligned to N * sizeof(T), at most 16 bytes each)
template <typename T, int N>
struct alignas(N * sizeof(T) > 16 ? 16 : N * sizeof(T)) Pack {
    T v[N];
};

// ------------------------------------------------- norm + rotary positions
// y = x * rsqrt(mean(x^2) + eps) * w over the d channels of one head, then pair
// i of the first `rot` channels, (y_i, y_{i + rot/2}), turned by the angle
// pos[axis(i)] * f_i. The angle is a product of a position and a frequency:
// formed in 64 bits in whole turns, its fraction is exact to 2^-25 turns in 32
// bits whatever the position, so sin and cos are 32-bit functions of the
// fraction alone.
struct RopeArgs {
    HeadsIn q, k;
    void *q_out, *k_out;
    const int* pos;
    const float *qw, *kw;
    float eps, inv_d;
    int tokens, n_q, n_kv, d, rot;
    int per_token;   // warps that share a token
    RopeTable tab;
};

constexpr int kRopeThreads = 256;

// cos and sin of the angle of a pair whose frequency is `turns` (in whole turns)
__device__ __forceinline__ float2 rope_turn(int pos, double turns) {
    const double turn = (double)pos * turns;
    float s, c;
    sincospif(2.0f * (float)(turn - rint(turn)), &s, &c);
    return make_float2(c, s);
}

// four elements as two pairs of floats
__device__ __forceinline__ void load_quad(const float* p, float2 (&x)[2]) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = make_float2(v.x, v.y);
    x[1] = make_float2(v.z, v.w);
}
template <typename T>
struct Quad {   // 16-bit
    uint2 w;
    __device__ __forceinline__ float2 lo() const { return unpack2(w.x, T{}); }
    __device__ __forceinline__ float2 hi() const { return unpack2(w.y, T{}); }
    __device__ __forceinline__ static Quad of(float2 a, float2 b) {
        Quad q;
        q.w = make_uint2(pack2<T>(a.x, a.y), pack2<T>(b.x, b.y));
        return q;
    }
};
template <>
struct Quad<float> {
    float4 w;
    __device__ __forceinline__ float2 lo() const { return make_float2(w.x, w.y); }
    __device__ __forceinline__ float2 hi() const { return make_float2(w.z, w.w); }
    __device__ __forceinline__ static Quad of(float2 a, float2 b) {
        Quad q;
        q.w = make_float4(a.x, a.y, b.x, b.y);
        return q;
    }
};

// A warp has one token (or a share of its heads). GS lanes (the power of two >= d
// / 8) have a row; lane l the two quads of channels [c0, c0 + 4) and [c1, c1 + 4)
// that pair up with each other, so a row is rotated without exchanging values and
// a lane's four sines and cosines, times the norm's weights, serve every head
// from registers: inv * (x0 (w0 cos) - x1 (w1 sin)), two channels an instruction
// (f32x2). What bounds it besides HBM is issue: 190 instructions a row at one
// channel an instruction (32 us at 4099 tokens of 40 heads of 128), hence D, the
// usual widths with every channel turned, known to the compiler (0: any). kRows
// rows a lane are loaded before the first is used.
template <typename TI, typename TO, int D>
__global__ void __launch_bounds__(kRopeThreads, D ? 4 : 2)
qk_norm_rope_kernel(const __grid_constant__ RopeArgs a, int gs_any) {
    __shared__ double turns[kMaxPairs];
    __shared__ unsigned char axis[kMaxPairs];
    const int gs = D ? D / 8 : gs_any, d = D ? D : a.d, rot = D ? D : a.rot;
    const int wid = blockIdx.x * (kRopeThreads / 32) + (threadIdx.x >> 5);
    const int t = wid / a.per_token, share = wid - t * a.per_token;
    const int lane = threadIdx.x & (gs - 1), sub = (threadIdx.x & 31) / gs, n_sub = 32 / gs;
    for (int i = threadIdx.x; i < rot / 2; i += kRopeThreads) {   // once a CTA: lanes index it apart
        turns[i] = a.tab.turns[i];
        axis[i] = a.tab.axis[i];
    }
    __syncthreads();
    pdl_trigger();
    pdl_wait();
    if (t >= a.tokens) return;
    const bool on = D || lane < d / 8, turned = D || lane < rot / 8;
    const int c0 = turned ? 4 * lane : 8 * lane, c1 = D ? c0 + D / 2 : turned ? rot / 2 + 4 * lane : 8 * lane + 4;
    constexpr int kRows = sizeof(TI) == 4 ? 3 : 4;
    // the groups of a warp have the same pairs: each works out its share of the
    // four (two groups: pairs sub, sub + 2; four and more: one each) and hands it on
    float2 co[2], si[2];
    const int shared = min(n_sub, 4);
    #pragma unroll
    for (int e = 0; e < 4; ++e) {
        float2 v = make_float2(1.f, 0.f);
        if (e * shared < 4) {
            const int pair = 4 * lane + e * shared + (sub & (shared - 1));
            if (turned && on) v = rope_turn(a.pos[(long long)axis[pair] * a.tokens + t], turns[pair]);
        }
        if (e & 1) { co[e >> 1].y = v.x; si[e >> 1].y = v.y; }
        else { co[e >> 1].x = v.x; si[e >> 1].x = v.y; }
    }
    if (shared == 2) {
        const float2 c = co[0], s = si[0];
        co[0] = make_float2(__shfl_sync(0xffffffffu, c.x, lane), __shfl_sync(0xffffffffu, c.x, lane + gs));
        co[1] = make_float2(__shfl_sync(0xffffffffu, c.y, lane), __shfl_sync(0xffffffffu, c.y, lane + gs));
        si[0] = make_float2(__shfl_sync(0xffffffffu, s.x, lane), __shfl_sync(0xffffffffu, s.x, lane + gs));
        si[1] = make_float2(__shfl_sync(0xffffffffu, s.y, lane), __shfl_sync(0xffffffffu, s.y, lane + gs));
    } else if (shared == 4) {
        const float c = co[0].x, s = si[0].x;
        co[0] = make_float2(__shfl_sync(0xffffffffu, c, lane), __shfl_sync(0xffffffffu, c, lane + gs));
        co[1] = make_float2(__shfl_sync(0xffffffffu, c, lane + 2 * gs), __shfl_sync(0xffffffffu, c, lane + 3 * gs));
        si[0] = make_float2(__shfl_sync(0xffffffffu, s, lane), __shfl_sync(0xffffffffu, s, lane + gs));
        si[1] = make_float2(__shfl_sync(0xffffffffu, s, lane + 2 * gs), __shfl_sync(0xffffffffu, s, lane + 3 * gs));
    }
    const int step = a.per_token * n_sub;
    #pragma unroll 1
    for (int part = 0; part < 2; ++part) {
        const int nh = part ? a.n_kv : a.n_q;
        if (nh == 0) continue;
        const HeadsIn& in = part ? a.k : a.q;
        const TI* src = static_cast<const TI*>(in.p) + (long long)t * in.tok + c0;
        TO* dst = static_cast<TO*>(part ? a.k_out : a.q_out) + (long long)t * nh * d + c0;
        const int head = (int)in.head;
        const float* wp = part ? a.kw : a.qw;
        float2 w0[2], w1[2];
        w0[0] = w0[1] = w1[0] = w1[1] = make_float2(1.f, 1.f);
        if (wp && on) {
            load_quad(wp + c0, w0);
            load_quad(wp + c1, w1);
        }
        // x0 -> x0 * f00 + x1 * f01, x1 -> x1 * f11 + x0 * f10
        float2 f00[2], f01[2], f10[2], f11[2];
        #pragma unroll
        for (int e = 0; e < 2; ++e) {
            f00[e] = mul2(w0[e], co[e]);
            f01[e] = mul2(w1[e], make_float2(-si[e].x, -si[e].y));
            f10[e] = mul2(w0[e], si[e]);
            f11[e] = mul2(w1[e], co[e]);
        }
        for (int h0 = share * n_sub; h0 < nh; h0 += kRows * step) {
            Quad<TI> x[kRows][2];
            #pragma unroll
            for (int u = 0; u < kRows; ++u) {   // past the last head: the last one again
                const TI* p = src + (long long)min(h0 + sub + u * step, nh - 1) * head;
                if (D || on) {
                    x[u][0] = *reinterpret_cast<const Quad<TI>*>(p);
                    x[u][1] = *reinterpret_cast<const Quad<TI>*>(p + (c1 - c0));
                } else {
                    x[u][0] = x[u][1] = Quad<TI>{};
                }
            }
            #pragma unroll
            for (int u = 0; u < kRows; ++u) {
                const float2 y0[2] = {x[u][0].lo(), x[u][0].hi()}, y1[2] = {x[u][1].lo(), x[u][1].hi()};
                float2 inv2 = make_float2(1.f, 1.f);
                if (wp) {
                    const float2 s2 = fma2(y0[0], y0[0], fma2(y0[1], y0[1], fma2(y1[0], y1[0], mul2(y1[1], y1[1]))));
                    float ss = s2.x + s2.y;
                    #pragma unroll
                    for (int o = 16; o > 0; o >>= 1)
                        if (o < gs) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                    inv2.x = inv2.y = rsqrtf(fmaf(ss, a.inv_d, a.eps));
                }
                float2 r0[2], r1[2];
                #pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (turned) {
                        r0[e] = mul2(fma2(y0[e], f00[e], mul2(y1[e], f01[e])), inv2);
                        r1[e] = mul2(fma2(y1[e], f11[e], mul2(y0[e], f10[e])), inv2);
                    } else {
                        r0[e] = mul2(mul2(y0[e], w0[e]), inv2);
                        r1[e] = mul2(mul2(y1[e], w1[e]), inv2);
                    }
                }
                if (h0 + sub + u * step < nh && on) {
                    TO* p = dst + (h0 + sub + u * step) * d;
                    *reinterpret_cast<Quad<TO>*>(p) = Quad<TO>::of(r0[0], r0[1]);
                    *reinterpret_cast<Quad<TO>*>(p + (c1 - c0)) = Quad<TO>::of(r1[0], r1[1]);
                }
            }
        }
    }
}

// The same for head widths, rotated widths, strides or addresses that the
// quads do not fit: one warp per row, single elements.
template <typename TI, typename TO>
__global__ void __launch_bounds__(kRopeThreads)
qk_norm_rope_any_kernel(const __grid_constant__ RopeArgs a) {
    extern __shared__ float2 cs[];
    const int t0 = blockIdx.x, lane = threadIdx.x & 31;
    pdl_trigger();
    pdl_wait();
    const int nh = a.n_q + a.n_kv, pairs = a.rot / 2;
    for (int p = threadIdx.x; p < pairs; p += kRopeThreads)
        cs[p] = rope_turn(a.pos[(long long)a.tab.axis[p] * a.tokens + t0], a.tab.turns[p]);
    __syncthreads();
    for (int h = threadIdx.x >> 5; h < nh; h += kRopeThreads / 32) {
        const bool isq = h < a.n_q;
        const TI* src = isq ? static_cast<const TI*>(a.q.p) + (long long)t0 * a.q.tok + (long long)h * a.q.head
                            : static_cast<const TI*>(a.k.p) + (long long)t0 * a.k.tok + (long long)(h - a.n_q) * a.k.head;
        TO* dst = isq ? static_cast<TO*>(a.q_out) + ((long long)t0 * a.n_q + h) * a.d
                      : static_cast<TO*>(a.k_out) + ((long long)t0 * a.n_kv + (h - a.n_q)) * a.d;
        const float* w = isq ? a.qw : a.kw;
        float inv = 1.0f;
        if (w) {
            float ss = 0.f;
            for (int c = lane; c < a.d; c += 32) {
                const float v = to_f(src[c]);
                ss = fmaf(v, v, ss);
            }
            for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            inv = rsqrtf(fmaf(ss, a.inv_d, a.eps));
        }
        for (int p = lane; p < pairs; p += 32) {
            float u0 = to_f(src[p]), u1 = to_f(src[p + pairs]);
            if (w) {
                u0 *= inv * w[p];
                u1 *= inv * w[p + pairs];
            }
            const float2 c = cs[p];
            dst[p] = from_f<TO>(fmaf(u0, c.x, -(u1 * c.y)));
            dst[p + pairs] = from_f<TO>(fmaf(u1, c.x, u0 * c.y));
        }
        for (int c = a.rot + lane; c < a.d; c += 32) {
            const float u = to_f(src[c]);
            dst[c] = from_f<TO>(w ? u * (inv * w[c]) : u);
        }
    }
}

bool heads_aligned(const HeadsIn& h, size_t esize, int elems) {
    return reinterpret_cast<uintptr_t>(h.p) % (esize * elems) == 0 && h.tok % elems == 0 && h.head % elems == 0;
}

size_t type_size(int type) { return type == kF32 ? 4 : 2; }

}  // namespace

cudaError_t qk_norm_rope(void* q_out, void* k_out, int out_type, const HeadsIn& q, const HeadsIn& k, int in_type,
                         const int* pos, const RopeTable& tab, int rot, const float* qw, const float* kw, float eps,
                         int tokens, int n_q, int n_kv, int d, cudaStream_t st) {
    if (tokens <= 0) return cudaSuccess;
    RopeArgs a{q, k, q_out, k_out, pos, qw, kw, eps, 1.0f / (float)d, tokens, n_q, n_kv, d, rot, 1, tab};
    const size_t os = type_size(out_type);
    const bool quads = d % 8 == 0 && rot % 8 == 0 && heads_aligned(q, type_size(in_type), 4) &&
                       (n_kv == 0 || heads_aligned(k, type_size(in_type), 4)) && std::abs(q.head) < INT_MAX &&
                       (n_kv == 0 || std::abs(k.head) < INT_MAX) &&
                       (reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(k_out)) % (4 * os) == 0 &&
                       (reinterpret_cast<uintptr_t>(qw) | reinterpret_cast<uintptr_t>(kw)) % 16 == 0;
    int gs = 1;
    while (gs < d / 8) gs *= 2;
    // few tokens: their heads are shared out, down to one round of rows a warp,
    // until the warps fill the SMs
    const int rounds = (std::max(n_q, n_kv) * gs + 31) / 32;
    while (a.per_token < rounds && (long long)tokens * a.per_token < 148 * 16) a.per_token *= 2;
    const long long warps = (long long)tokens * a.per_token;
    if (warps > INT_MAX) return cudaErrorInvalidValue;
    const cudaError_t e = by_type(in_type, [&](auto ti) {
        return by_type(out_type, [&](auto to) {
            using TI = decltype(ti);
            using TO = decltype(to);
            if (!quads)
                return launch_k(qk_norm_rope_any_kernel<TI, TO>, dim3(tokens), dim3(kRopeThreads),
                                sizeof(float2) * (rot / 2), st, a);
            const dim3 grid((unsigned)((warps + 7) / 8));
            const auto kernel = rot == d && d == 128 ? qk_norm_rope_kernel<TI, TO, 128>
                              : rot == d && d == 64  ? qk_norm_rope_kernel<TI, TO, 64>
                                                     : qk_norm_rope_kernel<TI, TO, 0>;
            return launch_k(kernel, grid, dim3(kRopeThreads), 0, st, a, gs);
        });
    });
    return e != cudaSuccess ? e : cudaGetLastError();
}

// ------------------------------------------------------------- 4-bit cache
// One group = 32 channels of one token and head: m = fp16(min), s = fp16((max -
// min) / 15), code = rne((x - m) / s) in 0..15; value = code * s + m. Each step
// is one correctly rounded 32-bit operation, so the codes are those of any
// other IEEE implementation. m and s are the values as stored (16 bits each: 1
// bit a channel for both; the codes make up for their rounding, which moves the
// group's range by at most 2^-11 of its ends). A NaN or an infinity in a group
// makes its s and m NaN: the group then reads as NaN instead of hiding it.
//
// Blocks hold 16 tokens x one head, laid out as the fragments of the matrix
// instructions that read them (NG = d / 32 groups; token t = 8 j + n for keys,
// t = 8 j + 2 quad + e for values and scales):
//   key codes    [j][n][quad][g]  32-bit words, nibble i = channel 32 g + 8 quad + i
//   key scales   [quad][g][j][e]  fp16
//   key minima   [n][j][g]        fp16
//   value codes  [j][n][quad][g]  32-bit words, nibble 4 e + i = channel 32 g + 4 n + i
//   value scales [quad][g][j][e]  fp16
//   value minima [quad][g][j][e]  fp16
struct Kv4At {
    uint8_t* block;
    int t;         // token in the block
    int by_quad;   // index of its scale for this lane's group
};

__device__ __forceinline__ Kv4At kv4_at(const Kv4Cache& c, long long slot, int head, int ng, int g) {
    // pages are powers of two of at least a block, and at most 2^31 slots in all
    const int shift = 31 - __clz(c.page), s = (int)slot;
    const int blk = (s & (c.page - 1)) / kKv4Block;
    Kv4At r;
    r.t = s % kKv4Block;
    r.block = c.p + ((((long long)(s >> shift) * c.n_kv + head) << (shift - 4)) + blk) * (20ll * c.d);
    r.by_quad = ((((r.t & 7) >> 1) * ng + g) * 2 + (r.t >> 3)) * 2 + (r.t & 1);
    return r;
}

// where a lane's 8 channels 32 g + 8 quad + i lie: a word of key codes; the
// halves of two words of value codes (channels 4 (2 quad) .. and 4 (2 quad + 1) ..),
// 4 ng words apart
__device__ __forceinline__ uint32_t* kv4_key_code(const Kv4At& at, int ng, int g, int quad) {
    return reinterpret_cast<uint32_t*>(at.block) + (at.t * 4 + quad) * ng + g;
}
__device__ __forceinline__ uint16_t* kv4_value_code(const Kv4At& at, int ng, int g, int quad) {
    return reinterpret_cast<uint16_t*>(at.block + 320 * ng) +
           ((((at.t >> 3) * 8 + 2 * quad) * 4 + ((at.t & 7) >> 1)) * ng + g) * 2 + (at.t & 1);
}
__device__ __forceinline__ __half* kv4_key_min(const Kv4At& at, int ng, int g) {
    return reinterpret_cast<__half*>(at.block + 288 * ng) + ((at.t & 7) * 2 + (at.t >> 3)) * ng + g;
}
// scales of the keys at byte 256 ng, of the values at 576 ng, minima of the values at 608 ng
__device__ __forceinline__ __half* kv4_by_quad(const Kv4At& at, int byte) {
    return reinterpret_cast<__half*>(at.block + byte) + at.by_quad;
}

// codes of 8 channels (one nibble each) and the group's s, m; the group is
// spread over the 4 lanes of a quad. The quotient (x - m) / s is first taken as
// one saturated fma with 1 / (15 s): good to 2^-17 + |m / s| 2^-21 of a step.
// Only where that leaves the nearest code open (a step's middle is that near:
// one bf16 value in 1200, one lane in 170) is it divided.
__device__ __forceinline__ uint32_t kv4_quantize(const float (&x)[8], __half& s, __half& m) {
    float lo = min_nan(min_nan(x[0], x[1], x[2]), min_nan(x[3], x[4], x[5]), min_nan(x[6], x[7], x[7]));
    float hi = max_nan(max_nan(x[0], x[1], x[2]), max_nan(x[3], x[4], x[5]), max_nan(x[6], x[7], x[7]));
    {
        const float a = __shfl_xor_sync(0xffffffffu, lo, 1), b = __shfl_xor_sync(0xffffffffu, lo, 2);
        const float c = __shfl_xor_sync(0xffffffffu, lo, 3);
        lo = min_nan(lo, a, min_nan(b, c, c));
        const float d = __shfl_xor_sync(0xffffffffu, hi, 1), e = __shfl_xor_sync(0xffffffffu, hi, 2);
        const float f = __shfl_xor_sync(0xffffffffu, hi, 3);
        hi = max_nan(hi, d, max_nan(e, f, f));
    }
    const bool bad = !(fabsf(lo) <= 3.402823466e38f && fabsf(hi) <= 3.402823466e38f);
    lo = fminf(fmaxf(lo, -65504.0f), 65504.0f);
    hi = fminf(fmaxf(hi, -65504.0f), 65504.0f);
    s = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
    m = __float2half_rn(lo);
    if (bad) s = m = __ushort_as_half(0x7fff);
    const float sf = __half2float(s), mf = __half2float(m);
    const float inv = sf > 0.0f ? __fdividef(1.0f, 15.0f * sf) : 0.0f, off = -mf * inv;
    // the code in the low bits of 1.5 * 2^23 + code
    uint32_t w = 0;
    float nearest = 0.f;   // the largest distance of a quotient from its code
    #pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float2 f = make_float2(__saturatef(fmaf(x[i], inv, off)), __saturatef(fmaf(x[i + 1], inv, off)));
        const float2 k15 = make_float2(15.f, 15.f), kr = make_float2(kRoundConst, kRoundConst);
        const float2 u = fma2(f, k15, kr);
        const float2 d = fma2(f, k15, fma2(u, make_float2(-1.f, -1.f), kr));
        nearest = fmaxf(nearest, fmaxf(fabsf(d.x), fabsf(d.y)));
        w += __float_as_uint(u.x) << (4 * i);
        w += __float_as_uint(u.y) << (4 * i + 4);
    }
    w -= 0x3F400000u;   // what the eight shifted 0x4B400000 (1.5 * 2^23) add up to
    const float open = 0.5f - 1.0f / 65536.0f - fabsf(off) * (15.0f / 2097152.0f);
    if (!(nearest <= open)) {   // NaN, too: its codes are 0 either way
        uint32_t which = 0;
        #pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float f = __saturatef(fmaf(x[i], inv, off));
            const float d = fmaf(f, 15.0f, kRoundConst - fmaf(f, 15.0f, kRoundConst));
            which |= fabsf(d) > open ? 1u << i : 0u;
        }
        while (which) {
            const int i = __ffs(which) - 1;
            which &= which - 1;
            float xi = x[0];
            #pragma unroll
            for (int y = 1; y < 8; ++y) xi = i == y ? x[y] : xi;
            const float c = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(xi, mf), sf)), 0.0f), 15.0f);
            w = (w & ~(15u << (4 * i))) | (uint32_t)(int)c << (4 * i);
        }
    }
    return w;
}

constexpr int kKv4Threads = 256;

template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, float (&x)[8]) {
    if (vec) {
        constexpr int N = sizeof(T) == 4 ? 4 : 8;
        #pragma unroll
        for (int h = 0; h < 8 / N; ++h) {
            const Pack<T, N> v = *reinterpret_cast<const Pack<T, N>*>(p + h * N);
            #pragma unroll
            for (int i = 0; i < N; ++i) x[h * N + i] = to_f(v.v[i]);
        }
    } else {
        #pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f(p[i]);
    }
}

// 8 channels of each lane to p + 8 * lane (whole warp). fp32: neighbouring lanes
// trade halves first, so that each store of the warp is one run of bytes.
template <typename T>
__device__ __forceinline__ void store8(T* p, float (&x)[8], bool on) {
    if constexpr (sizeof(T) == 4) {
        const bool odd = threadIdx.x & 1;
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float y = __shfl_xor_sync(0xffffffffu, odd ? x[i] : x[i + 4], 1);
            if (odd) x[i] = y;
            else x[i + 4] = y;
        }
        // even: its 0..3 and the odd lane's 0..3; odd: the even lane's 4..7 and its 4..7
        if (on) {
            *reinterpret_cast<float4*>(p + (odd ? -4 : 0)) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4*>(p + (odd ? 4 : 8)) = make_float4(x[4], x[5], x[6], x[7]);
        }
    } else if (on) {
        Pack<T, 8> v;
        #pragma unroll
        for (int i = 0; i < 8; ++i) v.v[i] = from_f<T>(x[i]);
        *reinterpret_cast<Pack<T, 8>*>(p) = v;
    }
}

// One lane = 8 channels of the key and of the value of one token and head; 4 NG
// lanes a row. Rows run over the tokens first, so that a warp writes both halves
// of a value word and whole sectors of codes when neighbouring tokens have
// neighbouring slots.
template <typename T, int NG>
__global__ void __launch_bounds__(kKv4Threads)
kv4_append_kernel(Kv4Cache c, HeadsIn k, HeadsIn v, const long long* slots, int tokens, int vec) {
    pdl_trigger();
    pdl_wait();
    const long long row = ((long long)blockIdx.x * kKv4Threads + threadIdx.x) / (4 * NG);
    const int l = threadIdx.x % (4 * NG), g = l >> 2, quad = l & 3, head = blockIdx.y;
    const bool on = row < tokens;
    const long long slot = on ? slots[row] : -1;
    const bool in = slot >= 0 && slot < c.n_pages * c.page;
    if (on && slot >= c.n_pages * c.page) record_status(kStatusBadShape);
    float xk[8] = {}, xv[8] = {};
    if (on) {   // not waiting for the slot
        load8(static_cast<const T*>(k.p) + row * k.tok + head * k.head + 8 * l, vec, xk);
        load8(static_cast<const T*>(v.p) + row * v.tok + head * v.head + 8 * l, vec, xv);
    }
    __half ks, km, vs, vm;
    const uint32_t wk = kv4_quantize(xk, ks, km), wv = kv4_quantize(xv, vs, vm);
    if (!in) return;
    const Kv4At at = kv4_at(c, slot, head, NG, g);
    *kv4_key_code(at, NG, g, quad) = wk;
    uint16_t* vc = kv4_value_code(at, NG, g, quad);
    vc[0] = (uint16_t)wv;
    vc[8 * NG] = (uint16_t)(wv >> 16);
    // one lane of the group writes each of its four numbers
    __half* p = quad == 0 ? kv4_by_quad(at, 256 * NG) : quad == 1 ? kv4_key_min(at, NG, g)
              : kv4_by_quad(at, quad == 2 ? 576 * NG : 608 * NG);
    *p = quad == 0 ? ks : quad == 1 ? km : quad == 2 ? vs : vm;
}

template <typename T, int NG>
__global__ void __launch_bounds__(kKv4Threads)
kv4_read_kernel(Kv4Cache c, T* k_out, T* v_out, const long long* slots, int tokens) {
    pdl_trigger();
    pdl_wait();
    const long long row = ((long long)blockIdx.x * kKv4Threads + threadIdx.x) / (4 * NG);
    const int l = threadIdx.x % (4 * NG), g = l >> 2, quad = l & 3, head = blockIdx.y;
    const bool on = row < tokens;
    const long long slot = on ? slots[row] : -1;
    float xk[8] = {}, xv[8] = {};
    if (slot >= c.n_pages * c.page) record_status(kStatusBadShape);
    if (slot >= 0 && slot < c.n_pages * c.page) {
        const Kv4At at = kv4_at(c, slot, head, NG, g);
        const uint16_t* vc = kv4_value_code(at, NG, g, quad);
        const uint32_t wk = *kv4_key_code(at, NG, g, quad), wv = vc[0] | (uint32_t)vc[8 * NG] << 16;
        const float ks = __half2float(*kv4_by_quad(at, 256 * NG)), km = __half2float(*kv4_key_min(at, NG, g));
        const float vs = __half2float(*kv4_by_quad(at, 576 * NG)), vm = __half2float(*kv4_by_quad(at, 608 * NG));
        #pragma unroll
        for (int e = 0; e < 8; ++e) {
            xk[e] = fmaf(i2f_small((wk >> (4 * e)) & 15u), ks, km);
            xv[e] = fmaf(i2f_small((wv >> (4 * e)) & 15u), vs, vm);
        }
    }
    const long long at = (row * c.n_kv + head) * (32 * NG) + 8 * l;
    store8(k_out + at, xk, on);
    store8(v_out + at, xv, on);
}

cudaError_t kv4_append(const Kv4Cache& c, const HeadsIn& k, const HeadsIn& v, int type, const long long* slots,
                       int tokens, cudaStream_t st) {
    if (tokens <= 0) return cudaSuccess;
    const int n = type == kF32 ? 4 : 8;
    const int vec = heads_aligned(k, type_size(type), n) && heads_aligned(v, type_size(type), n);
    const long long blocks = ((long long)tokens * (c.d / 8) + kKv4Threads - 1) / kKv4Threads;
    const cudaError_t e = by_type(type, [&](auto t) {
        using T = decltype(t);
        return launch_k(c.d == 128 ? kv4_append_kernel<T, 4> : kv4_append_kernel<T, 2>, dim3((unsigned)blocks, c.n_kv),
                        dim3(kKv4Threads), 0, st, c, k, v, slots, tokens, vec);
    });
    return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t kv4_read(const Kv4Cache& c, void* k_out, void* v_out, int type, const long long* slots, int tokens,
                     cudaStream_t st) {
    if (tokens <= 0) return cudaSuccess;
    const long long blocks = ((long long)tokens * (c.d / 8) + kKv4Threads - 1) / kKv4Threads;
    const cudaError_t e = by_type(type, [&](auto t) {
        using T = decltype(t);
        return launch_k(c.d == 128 ? kv4_read_kernel<T, 4> : kv4_read_kernel<T, 2>, dim3((unsigned)blocks, c.n_kv),
                        dim3(kKv4Threads), 0, st, c, static_cast<T*>(k_out), static_cast<T*>(v_out), slots, tokens);
    });
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace vsb

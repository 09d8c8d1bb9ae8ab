// Head norms with multi-axis rotary positions, and the append / read operators
// of the paged 4-bit cache. All of them move each value once; what bounds them
// is HBM at prompt sizes and the launch at single tokens.
#include "serve_ops.h"
#include "launch.cuh"
#include "sm100.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>

namespace vsb {

namespace {

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// N consecutive elements as one access (p aligned to N * sizeof(T), at most 16 bytes each)
template <typename T, int N>
struct alignas(N * sizeof(T) > 16 ? 16 : N * sizeof(T)) Pack {
    T v[N];
};

template <typename F>
cudaError_t by_type(int type, F&& f) {
    switch (type) {
        case kF32: return f(float{});
        case kF16: return f(__half{});
        case kBF16: return f(__nv_bfloat16{});
    }
    return cudaErrorInvalidValue;
}

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

// A warp has one token (or a share of its heads). GS lanes (the power of two >= d
// / 8) have a row; lane l the two quads of channels [c0, c0 + 4) and [c1, c1 + 4)
// that pair up with each other, so a row is rotated without exchanging values and
// a lane's four sines and cosines, in registers, serve every head. kRows rows a
// lane are loaded before the first is used.
template <typename TI, typename TO>
__global__ void __launch_bounds__(kRopeThreads)
qk_norm_rope_kernel(const __grid_constant__ RopeArgs a, int gs) {
    __shared__ double turns[kMaxPairs];
    __shared__ unsigned char axis[kMaxPairs];
    const int wid = blockIdx.x * (kRopeThreads / 32) + (threadIdx.x >> 5);
    const int t = wid / a.per_token, share = wid - t * a.per_token;
    const int lane = threadIdx.x & (gs - 1), sub = (threadIdx.x & 31) / gs, n_sub = 32 / gs;
    for (int i = threadIdx.x; i < a.rot / 2; i += kRopeThreads) {   // once a CTA: lanes index it apart
        turns[i] = a.tab.turns[i];
        axis[i] = a.tab.axis[i];
    }
    __syncthreads();
    pdl_trigger();
    pdl_wait();
    if (t >= a.tokens) return;
    const bool on = lane < a.d / 8, turned = lane < a.rot / 8;
    const int c0 = turned ? 4 * lane : 8 * lane, c1 = turned ? a.rot / 2 + 4 * lane : 8 * lane + 4;
    using P = Pack<TI, 4>;
    using PO = Pack<TO, 4>;
    constexpr int kRows = 4;
    float2 cs[4];
    #pragma unroll
    for (int e = 0; e < 4; ++e)
        cs[e] = turned ? rope_turn(a.pos[(long long)axis[4 * lane + e] * a.tokens + t], turns[4 * lane + e])
                       : make_float2(1.f, 0.f);
    #pragma unroll 1
    for (int part = 0; part < 2; ++part) {
        const int nh = part ? a.n_kv : a.n_q;
        const HeadsIn& in = part ? a.k : a.q;
        const TI* src = static_cast<const TI*>(in.p) + (long long)t * in.tok;
        TO* dst = static_cast<TO*>(part ? a.k_out : a.q_out) + (long long)t * nh * a.d;
        const float* wp = part ? a.kw : a.qw;
        float4 w0 = make_float4(1.f, 1.f, 1.f, 1.f), w1 = w0;
        if (wp && on) {
            w0 = *reinterpret_cast<const float4*>(wp + c0);
            w1 = *reinterpret_cast<const float4*>(wp + c1);
        }
        for (int h0 = share * n_sub + sub; h0 - sub < nh; h0 += kRows * a.per_token * n_sub) {
            P x[kRows][2];
            #pragma unroll
            for (int u = 0; u < kRows; ++u) {
                const int h = h0 + u * a.per_token * n_sub;
                x[u][0] = x[u][1] = P{};
                if (h < nh && on) {
                    x[u][0] = *reinterpret_cast<const P*>(src + (long long)h * in.head + c0);
                    x[u][1] = *reinterpret_cast<const P*>(src + (long long)h * in.head + c1);
                }
            }
            #pragma unroll
            for (int u = 0; u < kRows; ++u) {
                const int h = h0 + u * a.per_token * n_sub;
                if (h - sub >= nh) break;   // the same for the whole warp
                float y0[4], y1[4];
                #pragma unroll
                for (int e = 0; e < 4; ++e) {
                    y0[e] = to_f(x[u][0].v[e]);
                    y1[e] = to_f(x[u][1].v[e]);
                }
                if (wp) {
                    float ss = 0.f;
                    #pragma unroll
                    for (int e = 0; e < 4; ++e) ss = fmaf(y0[e], y0[e], fmaf(y1[e], y1[e], ss));
                    for (int o = gs >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                    const float inv = rsqrtf(fmaf(ss, a.inv_d, a.eps));
                    y0[0] *= inv * w0.x; y0[1] *= inv * w0.y; y0[2] *= inv * w0.z; y0[3] *= inv * w0.w;
                    y1[0] *= inv * w1.x; y1[1] *= inv * w1.y; y1[2] *= inv * w1.z; y1[3] *= inv * w1.w;
                }
                PO o0, o1;
                #pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float u0 = y0[e], u1 = y1[e];
                    o0.v[e] = from_f<TO>(turned ? fmaf(u0, cs[e].x, -(u1 * cs[e].y)) : u0);
                    o1.v[e] = from_f<TO>(turned ? fmaf(u1, cs[e].x, u0 * cs[e].y) : u1);
                }
                if (h < nh && on) {
                    *reinterpret_cast<PO*>(dst + (long long)h * a.d + c0) = o0;
                    *reinterpret_cast<PO*>(dst + (long long)h * a.d + c1) = o1;
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
                       (n_kv == 0 || heads_aligned(k, type_size(in_type), 4)) &&
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
            return launch_k(qk_norm_rope_kernel<TI, TO>, dim3((unsigned)((warps + 7) / 8)), dim3(kRopeThreads), 0, st, a,
                            gs);
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
    uint32_t* kc;
    __half *ks, *km;
    uint16_t* vc;
    __half *vs, *vm;
};

// the block of slot (page, head), and the offsets of token t inside it for the
// group g and quad that a lane handles
__device__ __forceinline__ Kv4At kv4_at(const Kv4Cache& c, long long slot, int head, int g, int quad) {
    const int ng = c.d / kKv4Group;
    // pages are powers of two of at least a block, and at most 2^31 slots in all
    const int shift = 31 - __clz(c.page), page = (int)slot >> shift;
    const int blk = ((int)slot & (c.page - 1)) / kKv4Block, t = (int)slot % kKv4Block;
    uint8_t* b = c.p + ((((long long)page * c.n_kv + head) << (shift - 4)) + blk) * (20ll * c.d);
    const int j = t >> 3;
    const int by_quad = ((((t & 7) >> 1) * ng + g) * 2 + j) * 2 + (t & 1);
    Kv4At r;
    r.kc = reinterpret_cast<uint32_t*>(b) + (((j * 8 + (t & 7)) * 4 + quad) * ng + g);
    r.ks = reinterpret_cast<__half*>(b + 8 * c.d) + by_quad;
    r.km = reinterpret_cast<__half*>(b + 9 * c.d) + (((t & 7) * 2 + j) * ng + g);
    // n = 2 quad and 2 quad + 1: the second at + 4 * ng words
    r.vc = reinterpret_cast<uint16_t*>(b + 10 * c.d) + (((j * 8 + 2 * quad) * 4 + ((t & 7) >> 1)) * ng + g) * 2 + (t & 1);
    r.vs = reinterpret_cast<__half*>(b + 18 * c.d) + by_quad;
    r.vm = reinterpret_cast<__half*>(b + 19 * c.d) + by_quad;
    return r;
}

__device__ __forceinline__ float min_nan(float a, float b) {   // NaN if either is
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// codes of 8 channels (one nibble each) and the group's s, m; the group is
// spread over the 4 lanes of a quad. The quotient (x - m) / s is first taken as
// a product with 1 / (15 s), saturated to [0, 1]: good to 2^-20 of a step. Only
// where that leaves the nearest code open (a step's middle within 2^-16: one
// group in 500 of random values) is it divided.
__device__ __forceinline__ uint32_t kv4_quantize(const float (&x)[8], __half& s, __half& m) {
    float lo = x[0], hi = x[0];
    #pragma unroll
    for (int i = 1; i < 8; ++i) {
        lo = min_nan(lo, x[i]);
        hi = max_nan(hi, x[i]);
    }
    #pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const bool bad = !(fmaxf(fabsf(lo), fabsf(hi)) <= 3.402823466e38f) || lo != lo;
    lo = fminf(fmaxf(lo, -65504.0f), 65504.0f);
    hi = fminf(fmaxf(hi, -65504.0f), 65504.0f);
    s = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
    m = __float2half_rn(lo);
    if (bad) s = m = __ushort_as_half(0x7fff);
    const float sf = __half2float(s), mf = __half2float(m);
    const float inv = sf > 0.0f ? __fdividef(1.0f, 15.0f * sf) : 0.0f;
    // the code in the low bits of 1.5 * 2^23 + code
    uint32_t w = 0;
    float nearest = 0.f;   // the largest distance of a quotient from its code
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float f = __saturatef(__fsub_rn(x[i], mf) * inv);
        const float u = fmaf(f, 15.0f, kRoundConst);
        nearest = fmaxf(nearest, fabsf(fmaf(f, 15.0f, kRoundConst - u)));
        w += (__float_as_uint(u) - 0x4B400000u) << (4 * i);
    }
    if (nearest > 0.5f - 1.0f / 65536.0f) {
        w = 0;
        #pragma unroll 1
        for (int i = 0; i < 8; ++i) {
            float xi = x[0];
            #pragma unroll
            for (int y = 1; y < 8; ++y) xi = i == y ? x[y] : xi;
            const float c = sf > 0.0f ? rintf(__fdiv_rn(__fsub_rn(xi, mf), sf)) : 0.0f;
            w |= (uint32_t)(int)fminf(fmaxf(c, 0.0f), 15.0f) << (4 * i);
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

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    constexpr int N = sizeof(T) == 4 ? 4 : 8;
    #pragma unroll
    for (int h = 0; h < 8 / N; ++h) {
        Pack<T, N> v;
        #pragma unroll
        for (int i = 0; i < N; ++i) v.v[i] = from_f<T>(x[h * N + i]);
        *reinterpret_cast<Pack<T, N>*>(p + h * N) = v;
    }
}

// One lane = 8 channels of one token, head and of keys or values; d / 8 lanes a
// row. Rows run over the tokens first, so that a warp writes both halves of a
// value word and whole sectors of codes when neighbouring tokens have
// neighbouring slots.
template <typename T>
__global__ void __launch_bounds__(kKv4Threads)
kv4_append_kernel(Kv4Cache c, HeadsIn k, HeadsIn v, const long long* slots, int tokens, int vec) {
    pdl_trigger();
    pdl_wait();
    const int lanes = c.d == 128 ? 4 : 3;   // log2 of a row's
    const long long row = ((long long)blockIdx.x * kKv4Threads + threadIdx.x) >> lanes;
    const int l = threadIdx.x & ((1 << lanes) - 1), head = blockIdx.y;
    const bool on = row < tokens;
    const long long slot = on ? slots[row] : -1;
    const bool in = slot >= 0 && slot < c.n_pages * c.page;
    if (on && slot >= c.n_pages * c.page) record_status(kStatusBadShape);
    const T* src = blockIdx.z ? static_cast<const T*>(v.p) + row * v.tok + head * v.head
                              : static_cast<const T*>(k.p) + row * k.tok + head * k.head;
    float x[8] = {};
    if (in) load8(src + 8 * l, vec, x);
    __half s, m;
    const uint32_t w = kv4_quantize(x, s, m);
    if (!in) return;
    const Kv4At at = kv4_at(c, slot, head, l >> 2, l & 3);
    if (blockIdx.z == 0) {
        *at.kc = w;
        if ((l & 3) == 0) {
            *at.ks = s;
            *at.km = m;
        }
    } else {
        at.vc[0] = (uint16_t)w;
        at.vc[4 * (c.d / kKv4Group) * 2] = (uint16_t)(w >> 16);
        if ((l & 3) == 0) {
            *at.vs = s;
            *at.vm = m;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kKv4Threads)
kv4_read_kernel(Kv4Cache c, T* k_out, T* v_out, const long long* slots, int tokens) {
    pdl_trigger();
    pdl_wait();
    const int lanes = c.d == 128 ? 4 : 3;   // log2 of a row's
    const long long row = ((long long)blockIdx.x * kKv4Threads + threadIdx.x) >> lanes;
    const int l = threadIdx.x & ((1 << lanes) - 1), head = blockIdx.y;
    if (row >= tokens) return;
    const long long slot = slots[row];
    float x[8] = {};
    if (slot >= c.n_pages * c.page) record_status(kStatusBadShape);
    if (slot >= 0 && slot < c.n_pages * c.page) {
        const Kv4At at = kv4_at(c, slot, head, l >> 2, l & 3);
        const uint32_t w = blockIdx.z == 0 ? *at.kc : (uint32_t)at.vc[0] | (uint32_t)at.vc[8 * (c.d / kKv4Group)] << 16;
        const float s = __half2float(blockIdx.z == 0 ? *at.ks : *at.vs);
        const float m = __half2float(blockIdx.z == 0 ? *at.km : *at.vm);
        #pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = fmaf((float)((w >> (4 * e)) & 15u), s, m);
    }
    store8((blockIdx.z ? v_out : k_out) + (row * c.n_kv + head) * c.d + 8 * l, x);
}

cudaError_t kv4_append(const Kv4Cache& c, const HeadsIn& k, const HeadsIn& v, int type, const long long* slots,
                       int tokens, cudaStream_t st) {
    if (tokens <= 0) return cudaSuccess;
    const int n = type == kF32 ? 4 : 8;
    const int vec = heads_aligned(k, type_size(type), n) && heads_aligned(v, type_size(type), n);
    const long long blocks = ((long long)tokens * (c.d / 8) + kKv4Threads - 1) / kKv4Threads;
    const cudaError_t e = by_type(type, [&](auto t) {
        return launch_k(kv4_append_kernel<decltype(t)>, dim3((unsigned)blocks, c.n_kv, 2), dim3(kKv4Threads), 0, st, c,
                        k, v, slots, tokens, vec);
    });
    return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t kv4_read(const Kv4Cache& c, void* k_out, void* v_out, int type, const long long* slots, int tokens,
                     cudaStream_t st) {
    if (tokens <= 0) return cudaSuccess;
    const long long blocks = ((long long)tokens * (c.d / 8) + kKv4Threads - 1) / kKv4Threads;
    const cudaError_t e = by_type(type, [&](auto t) {
        using T = decltype(t);
        return launch_k(kv4_read_kernel<T>, dim3((unsigned)blocks, c.n_kv, 2), dim3(kKv4Threads), 0, st, c,
                        static_cast<T*>(k_out), static_cast<T*>(v_out), slots, tokens);
    });
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace vsb

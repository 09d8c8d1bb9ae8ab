// Attention over packed prompts: grouped heads, causal or dense, sequences of
// different lengths one after another in one array.
//
// One pass over the keys with the running maximum m and sum l of a softmax:
//   S = Q K^T;  P = 2^(c (S - m)), c = scale log2(e);  l += rowsum P;  O += P V
// both products on tcgen05 (128 x 64 x D and 128 x D x 64, accumulators in TMEM),
// P written back over S's columns as the A operand of the second one, so scores
// and weights never leave the SM. 16384 tokens, 32 heads over 8 of 128, causal:
// 1.76 to 2.04 ms by the card and its power cap, 1.08 to 1.25 PFLOP/s (64 to 75 %
// of a large library product's burst rate); a step of 64 keys takes the two tiles
// 1750 cycles, the tensor core 1400 of them, the rest is the softmax's
// instruction latency.
//
// A CTA has two 128-row tiles of one key head. A tile's rows are (query, head of
// the group) pairs, token-major: the keys of a group are loaded once for all of
// its heads, and a causal tile spans 128 / group tokens, which keeps what the
// mask throws away small. Warps: 0-3 and 4-7 the softmax of tile 0 and 1 (thread
// = row = TMEM lane), 8 and 9 issue the matrix products of tile 0 and 1, 10 the
// TMA loads of a ring of K and V tiles, 11 looks over the value tiles that are
// not seen in full.
//
// TMEM's 512 columns are full with two O tiles of 128 channels and 128 columns of
// scores for each: as two buffers of 64 keys, so that the products of a buffer
// run under the softmax of the other. (One buffer of 128 keys, the two tiles in
// turn, left the tensor core idle for half the time: a block's softmax, 2000
// cycles, and its products, 1400, followed one another.)
//
// m only follows the true maximum when it is more than 2^8 behind (P then stays
// below 2^8, or 2^14 with fp16's factor, inside bf16 and fp16): O is rescaled in TMEM that rarely, by
// the softmax threads themselves.
//
// A score that is NaN or +infinity makes its row NaN, and so do scores that are
// -infinity throughout. The exponentials need not carry that (the polynomial
// cannot): the row's maximum is taken so that a NaN stays, and l becomes NaN.
#include "serve_ops.h"
#include "gemm_i8.h"
#include "launch.cuh"
#include "serve_math.cuh"
#include "sm100.cuh"

#include <atomic>
#include <climits>
#include <type_traits>

namespace vsb {

namespace {

struct PromptArgs {
    HeadsIn q, k, v;
    void* out;
    const int *cu_q, *cu_k, *prefix;
    int n_seq, total_q, total_k, n_q, n_kv, d, causal, negate;
    float scale_log2;   // |scale| * log2(e)
    int gp, tile_tok;   // heads and tokens of a 128-row tile
};

// keys that query i of a sequence of lq queries and lk keys sees: [0, limit)
__device__ __forceinline__ int prompt_limit(const PromptArgs& a, int seq, int i, int lq, int lk) {
    int lim = a.causal ? min(max(lk - lq + i + 1, 0), lk) : lk;
    if (a.prefix) lim = max(lim, min(a.prefix[seq], lk));
    return lim;
}

// One row by one warp, one key at a time: the definition. It serves the rows
// whose tile holds a NaN or an infinity in a value that the mask hides from some
// of its rows (0 * NaN would reach them through the matrix product).
template <typename T>
__device__ __noinline__ void prompt_row(const PromptArgs& a, int row, int head, int k0, int lim) {
    const int lane = threadIdx.x & 31, kvh = head / (a.n_q / a.n_kv);
    float o[4] = {}, q[4] = {}, m = -INFINITY, l = 0.f;
    const T* qp = static_cast<const T*>(a.q.p) + (long long)row * a.q.tok + (long long)head * a.q.head;
    const float c = a.negate ? -a.scale_log2 : a.scale_log2;
    #pragma unroll
    for (int x = 0; x < 4; ++x)
        if (lane + 32 * x < a.d) q[x] = to_f(qp[lane + 32 * x]);
    for (int j = 0; j < lim; ++j) {
        const T* kp = static_cast<const T*>(a.k.p) + (long long)(k0 + j) * a.k.tok + (long long)kvh * a.k.head;
        const T* vp = static_cast<const T*>(a.v.p) + (long long)(k0 + j) * a.v.tok + (long long)kvh * a.v.head;
        float s = 0.f;
        #pragma unroll
        for (int x = 0; x < 4; ++x)
            if (lane + 32 * x < a.d) s = fmaf(q[x], to_f(kp[lane + 32 * x]), s);
        for (int y = 16; y > 0; y >>= 1) s += __shfl_xor_sync(0xffffffffu, s, y);
        s *= c;
        const float mn = fmaxf(m, s);
        // a score of -infinity weighs nothing; NaN and +infinity stay (inf - inf)
        const float alpha = m == -INFINITY ? 1.f : ex2(m - mn), w = s == -INFINITY ? 0.f : ex2(s - mn);
        m = mn;
        l = fmaf(l, alpha, w);
        #pragma unroll
        for (int x = 0; x < 4; ++x)
            if (lane + 32 * x < a.d) o[x] = fmaf(o[x], alpha, w * to_f(vp[lane + 32 * x]));
    }
    const float inv = lim > 0 ? 1.0f / l : 0.f;   // keys that all weigh nothing: 0 * infinity
    T* out = static_cast<T*>(a.out) + ((long long)row * a.n_q + head) * a.d;
    #pragma unroll
    for (int x = 0; x < 4; ++x)
        if (lane + 32 * x < a.d) out[lane + 32 * x] = from_f<T>(o[x] * inv);
}

constexpr int kPaThreads = 384, kPaRows = 128, kPaKeys = 128;   // keys of a ring tile
constexpr int kPaStep = 64;                                     // keys of a step of the softmax
// registers a thread: the softmax warpgroups take what the third one gives up
constexpr int kPaRegsSoftmax = 208, kPaRegsRest = 88, kPaRegsAtLaunch = (2 * kPaRegsSoftmax + kPaRegsRest) / 3;
constexpr uint32_t kPaBoxBytes = 128 * 128;   // 128 rows of 64 channels

__host__ __device__ constexpr int pa_stages(int D) { return D == 128 ? 5 : 8; }
constexpr size_t pa_smem(int D) { return 1024 + (size_t)(2 + pa_stages(D)) * (D / 64) * kPaBoxBytes + 512; }

// kind::f16 instruction descriptor: F32 accumulator, A and B both bf16 or both
// fp16, M = 128; b_mn: B is stored with its N index innermost
__host__ __device__ constexpr uint32_t idesc_f16(bool bf16, int N, bool b_mn, bool neg_a) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((neg_a ? 1u : 0u) << 13) |
           ((b_mn ? 1u : 0u) << 16) | (static_cast<uint32_t>(N >> 3) << 17) | (8u << 24);
}

__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}

// Descriptor of a V tile as the B operand with N (channels) innermost: rows of
// 64 channels (128 bytes, swizzled), 8-key groups 1024 bytes apart (SBO), blocks
// of 64 channels 16384 bytes apart (LBO).
__device__ __forceinline__ uint64_t sw128_mnmajor_desc(uint32_t saddr) {
    return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(kPaBoxBytes >> 4) << 16) |
           (static_cast<uint64_t>(1024u >> 4) << 32) | (static_cast<uint64_t>(1u) << 46) |
           (static_cast<uint64_t>(2u) << 61);
}

__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
        :: "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
           "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
           "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
           "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
        :: "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
           "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ bool elect_one() {   // one lane of a converged warp
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

template <int N>
__device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(N)); }
template <int N>
__device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(N)); }

// The registers of a tcgen05.ld are there once tmem_ld_wait() has returned: no
// use of them may be moved in front of it.
template <int N>
__device__ __forceinline__ void tmem_ready(uint32_t (&r)[N]) {
    #pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}

// 2^x for x in [-126, 127] on the FMA pipe: x = n + f, |f| <= 1/2, 2^f by the
// polynomial of least relative error (fitted to 2^f by Remez exchange: 2^-13.7 at
// degree 3, 2^-18.5 at degree 4), n added to the exponent. Below -126 it stays at
// 2^-126, which the weights' type rounds to nothing beside a row's largest.
template <bool FINE>
__device__ __forceinline__ float2 ex2_poly(float2 x) {
    x.x = fmaxf(x.x, -126.f);
    x.y = fmaxf(x.y, -126.f);
    const float2 big = make_float2(kRoundConst, kRoundConst), nbig = make_float2(-kRoundConst, -kRoundConst);
    const float2 t = add2(x, big);
    const float2 f = fma2(add2(t, nbig), make_float2(-1.f, -1.f), x);
    float2 p;
    if constexpr (FINE) {
        p = fma2(make_float2(0.00957010210f, 0.00957010210f), f, make_float2(0.0559178628f, 0.0559178628f));
        p = fma2(p, f, make_float2(0.240247443f, 0.240247443f));
        p = fma2(p, f, make_float2(0.693121791f, 0.693121791f));
        p = fma2(p, f, make_float2(0.999999285f, 0.999999285f));
    } else {
        p = fma2(make_float2(0.0551716685f, 0.0551716685f), f, make_float2(0.242611125f, 0.242611125f));
        p = fma2(p, f, make_float2(0.693260968f, 0.693260968f));
        p = fma2(p, f, make_float2(0.999928057f, 0.999928057f));
    }
    p.x = __int_as_float(__float_as_int(p.x) + (__float_as_int(t.x) << 23));
    p.y = __int_as_float(__float_as_int(p.y) + (__float_as_int(t.y) << 23));
    return p;
}

// of 8 pairs of weights, how many the FMA pipe makes: the SFUs alone are as long as the tensor core, the polynomial
// costs issue slots. Four runs each in turn, 32 heads over 8 of 128, 16384 tokens (median, range) and a ragged batch of
// 8: 0: 1885 us (1848..1973), 105; 2: 1821 (1801..1947), 102; 3: 1785 (1757..1830), 100.5; 4: 1811 (1810..1845), 102
constexpr int kPaPoly = 3;

// What a CTA works on: tile t has rows of queries [tok[t], tok[t] + n_tok[t])
// of the sequence and sees the first keys[t] of its lk keys. bad[t]: a value that
// the mask hides from some row, in a block that tile t multiplies, is not finite.
struct PromptJob {
    int seq, q0, lq, k0, lk, tok[2], n_tok[2], keys[2], bad[2];
};

template <typename T, int D>
__global__ void __launch_bounds__(kPaThreads, 1)
prompt_tc_kernel(const __grid_constant__ PromptArgs a, const __grid_constant__ CUtensorMap mq,
                 const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv) {
    constexpr bool kBf16 = sizeof(T) == 2 && !std::is_same<T, __half>::value;
    constexpr int kStages = pa_stages(D), kCB = D / 64, kPoly = kPaPoly;
    constexpr uint32_t kTile = kCB * kPaBoxBytes;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* sq = sm;                       // two Q tiles
    uint8_t* ring = sm + 2 * kTile;
    uint64_t* q_full = reinterpret_cast<uint64_t*>(ring + kStages * kTile);
    uint64_t* kv_full = q_full + 1;
    uint64_t* v_raw = kv_full + kStages;    // value tiles that warp 11 looks over first
    uint64_t* kv_empty = v_raw + kStages;   // [pair % 4]
    uint64_t* s_full = kv_empty + 4;        // [tile][buffer]
    uint64_t* p_full = s_full + 4;
    uint64_t* o_done = p_full + 4;          // the last output product of a tile
    uint64_t* o_prev = o_done + 2;          // the one before it
    uint32_t* tslot = reinterpret_cast<uint32_t*>(o_prev + 2);
    PromptJob* job = reinterpret_cast<PromptJob*>(tslot + 2);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int head_blocks = a.n_q / a.gp;
    const int hb = blockIdx.x % head_blocks;
    const int head0 = hb * a.gp, kvh = head0 / (a.n_q / a.n_kv);
    if (tid == 0) {
        mbar_init(q_full, 1);
        for (int i = 0; i < kStages; ++i) {
            mbar_init(kv_full + i, 1);
            mbar_init(v_raw + i, 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(s_full + i, 1);
            mbar_init(p_full + i, 4);
            mbar_init(kv_empty + i, 2);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(o_done + t, 1);
            mbar_init(o_prev + t, 1);
        }
        fence_mbar_init();
        tma_prefetch_desc(&mq);
        tma_prefetch_desc(&mk);
        tma_prefetch_desc(&mv);
    }
    if (warp == 8) tmem_alloc(tslot, 512);
    pdl_wait();
    if (warp == 0) {
        // the sequence this CTA's pair of tiles lies in: pairs are numbered by
        // sequence, and within one from its end, the rows with the most keys first
        int want = blockIdx.x / head_blocks, found = -1, at = 0, q0 = 0, lq = 0, k0 = 0, lk = 0;
        for (int s0 = 0; s0 < a.n_seq && found < 0; s0 += 32) {
            const int s = s0 + lane;
            int n = 0, qa = 0, qb = 0, ka = 0, kb = 0;
            if (s < a.n_seq) {
                qa = min(max(a.cu_q[s], 0), a.total_q);
                qb = min(max(a.cu_q[s + 1], qa), a.total_q);
                ka = min(max(a.cu_k[s], 0), a.total_k);
                kb = min(max(a.cu_k[s + 1], ka), a.total_k);
                n = (qb - qa + 2 * a.tile_tok - 1) / (2 * a.tile_tok);
            }
            int sum = n;
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += x;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, want < sum);
            if (hit) {
                const int l = __ffs(hit) - 1;
                found = s0 + l;
                at = __shfl_sync(0xffffffffu, sum, l) - 1 - want;   // pairs after this one
                q0 = __shfl_sync(0xffffffffu, qa, l);
                lq = __shfl_sync(0xffffffffu, qb, l) - q0;
                k0 = __shfl_sync(0xffffffffu, ka, l);
                lk = __shfl_sync(0xffffffffu, kb, l) - k0;
            } else {
                want -= __shfl_sync(0xffffffffu, sum, 31);
            }
        }
        if (lane == 0) {
            PromptJob j = {};
            j.seq = found;
            if (found >= 0) {
                j.q0 = q0;
                j.lq = lq;
                j.k0 = k0;
                j.lk = lk;
                for (int t = 0; t < 2; ++t) {
                    j.tok[t] = (2 * at + t) * a.tile_tok;
                    j.n_tok[t] = min(max(j.lq - j.tok[t], 0), a.tile_tok);
                    j.keys[t] = j.n_tok[t] > 0 ? prompt_limit(a, found, j.tok[t] + j.n_tok[t] - 1, j.lq, j.lk) : 0;
                }
            }
            *job = j;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_trigger();
    const uint32_t tmem = *tslot;
    const int seq = job->seq;
    const int nblk0 = (job->keys[0] + kPaKeys - 1) / kPaKeys, nblk1 = (job->keys[1] + kPaKeys - 1) / kPaKeys;
    const int nblk = max(nblk0, nblk1);
    const int nstep0 = (job->keys[0] + kPaStep - 1) / kPaStep, nstep1 = (job->keys[1] + kPaStep - 1) / kPaStep;

    // the fewest keys any row here sees: past them some weights are masked to 0
    const int clear_all = nblk > 0 ? prompt_limit(a, seq, job->n_tok[0] > 0 ? job->tok[0] : job->tok[1], job->lq, job->lk) : 0;
    const int masked0 = clear_all / kPaKeys;   // the first block that is not seen in full
    // masked value blocks go round the ring's stages with this period
    constexpr int kPeriod = kStages % 2 ? kStages : kStages / 2;

    if (warp >= 8) {
        regs_dec<kPaRegsRest>();
        if (warp == 10 && nblk > 0) {
            // ---- loads: Q tiles, then K and V of each block through the ring
            if (lane == 0) {
                mbar_arrive_expect_tx(q_full, (uint32_t)((nblk0 > 0) + (nblk1 > 0)) * kCB * 128u * (uint32_t)(a.gp * a.tile_tok));
                for (int t = 0; t < 2; ++t)
                    if ((t ? nblk1 : nblk0) > 0)
                        for (int c = 0; c < kCB; ++c)
                            tma_load_3d(sq + t * kTile + c * kPaBoxBytes, &mq, q_full, 64 * c, head0, job->q0 + job->tok[t]);
                int i = 0;
                for (; i < 2 * nblk; ++i) {
                    const int st = i % kStages;
                    if (i >= kStages) {
                        const int old = (i - kStages + 1) >> 1;   // the pair of the tile that was here
                        if (!mbar_wait(kv_empty + (old & 3), (uint32_t)(old >> 2) & 1u)) break;
                    }
                    uint64_t* bar = (i & 1) && (i >> 1) >= masked0 ? v_raw + st : kv_full + st;
                    mbar_arrive_expect_tx(bar, kTile);
                    for (int c = 0; c < kCB; ++c)
                        tma_load_3d(ring + st * kTile + c * kPaBoxBytes, (i & 1) ? &mv : &mk, bar, 64 * c, kvh,
                                    job->k0 + (i >> 1) * kPaKeys);
                }
                // every copy has landed before the CTA may leave (after a wait that gave up, too)
                const uint64_t until = globaltimer_ns() + kWaitLimitNs;
                mbar_wait_until(q_full, 0, until);
                for (int x = max(0, i - kStages); x < i; ++x) {
                    if ((x & 1) && (x >> 1) >= masked0)
                        mbar_wait_until(v_raw + x % kStages, (uint32_t)(((x >> 1) - masked0) / kPeriod) & 1u, until);
                    else
                        mbar_wait_until(kv_full + x % kStages, (uint32_t)(x / kStages) & 1u, until);
                }
            }
        } else if (warp == 11) {
            // ---- value blocks that some row does not see all of: 0 * v has to be 0. Rows past the
            // sequence become zeros; a NaN or an infinity in front of its end is left to the rows that
            // see it, and the others are done again one by one.
            for (int j = masked0; j < nblk; ++j) {
                const int st = (2 * j + 1) % kStages;
                if (!__all_sync(0xffffffffu, mbar_wait(v_raw + st, (uint32_t)((j - masked0) / kPeriod) & 1u))) break;
                uint8_t* vt = ring + st * kTile;
                const int valid = min(job->lk - j * kPaKeys, kPaKeys);
                // an infinity or a NaN has all exponent bits: the largest magnitude, as whole numbers, tells
                constexpr uint32_t kExp = kBf16 ? 0x7F80u : 0x7C00u;
                const int seen = max(clear_all - j * kPaKeys, 0);   // keys in front that every row sees
                uint32_t big = 0;
                for (int c = 0; c < kCB; ++c) {
                    uint4* tile = reinterpret_cast<uint4*>(vt + c * kPaBoxBytes);   // 8 to a key
                    #pragma unroll 8
                    for (int x = seen * 8 + lane; x < valid * 8; x += 32) {
                        const uint4 w = tile[x];
                        big = __vmaxu2(__vmaxu2(big, w.x & 0x7FFF7FFFu), __vmaxu2(w.y & 0x7FFF7FFFu, w.z & 0x7FFF7FFFu));
                        big = __vmaxu2(big, w.w & 0x7FFF7FFFu);
                    }
                    #pragma unroll 4
                    for (int x = valid * 8 + lane; x < kPaKeys * 8; x += 32) tile[x] = make_uint4(0u, 0u, 0u, 0u);
                }
                const bool bad = (big & 0xFFFFu) >= kExp || big >> 16 >= kExp;
                // for the tiles that multiply this block alone: the end of their products comes after this
                if (bad && j < nblk0) job->bad[0] = 1;
                if (bad && j < nblk1) job->bad[1] = 1;
                __threadfence_block();
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(kv_full + st);
            }
        } else if (warp < 10 && nblk > 0) {
            // ---- matrix products of tile t, by one elected thread. It has to be elect.sync around the whole
            // loop: the operands of a product are uniform registers, and behind `lane == 0` inside the loop
            // each product took 50 to 90 cycles to issue (64 to run). One commit a step: that of the scores
            // of step i + 2 also tells that the output product of step i, issued before them, is done.
            const int t = warp - 8, ns = t ? nstep1 : nstep0;
            constexpr uint32_t kPV = idesc_f16(kBf16, D, true, false);
            const uint32_t kQK = a.negate ? idesc_f16(kBf16, kPaStep, false, true) : idesc_f16(kBf16, kPaStep, false, false);
            const uint64_t dq = sw128_kmajor_desc(smem_u32(sq + t * kTile)), dk = sw128_kmajor_desc(smem_u32(ring));
            const uint64_t dv = sw128_mnmajor_desc(smem_u32(ring));
            const uint32_t tS = tmem + 128 * t, tO = tmem + 256 + 128 * t;
            auto there = [&](int i) { return mbar_wait(kv_full + i % kStages, (uint32_t)(i / kStages) & 1u); };
            // scores of step i (half of K tile i / 2) into buffer i % 2; one thread
            auto qk = [&](int i) {
                const int st = (i & ~1) % kStages;
                const uint64_t dks = dk + ((st * kTile + (i & 1) * (kPaStep * 128)) >> 4);
                #pragma unroll
                for (int k = 0; k < D / 16; ++k) {   // 32 bytes a step, 64 channels a box
                    const int off = ((k >> 2) * kPaBoxBytes + (k & 3) * 32) >> 4;
                    umma_f16_ss(tS + kPaStep * (i & 1), dq + off, dks + off, kQK, k > 0);
                }
                umma_commit(s_full + 2 * t + (i & 1));
            };
            if (elect_one()) {
                bool ok = ns > 0 && mbar_wait(q_full, 0) && there(0);
                tc_fence_after();
                if (ok) qk(0);
                if (ok && ns > 1) qk(1);
                for (int i = 0; i < ns && ok; ++i) {
                    const int iv = 2 * (i >> 1) + 1, sv = iv % kStages, b = i & 1;
                    ok = (b || (there(iv) && (i + 2 >= ns || there(iv + 1)))) &&
                         mbar_wait(p_full + 2 * t + b, (uint32_t)(i >> 1) & 1u);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t dvs = dv + ((sv * kTile + b * (kPaStep * 128)) >> 4);
                    #pragma unroll
                    for (int k = 0; k < kPaStep / 16; ++k)
                        umma_f16_ts(tO, tS + kPaStep * b + 8 * k, dvs + k * (2048 >> 4), kPV, i > 0 || k > 0);
                    if (i + 2 < ns) qk(i + 2);
                    else umma_commit((i == ns - 1 ? o_done : o_prev) + t);
                }
            }
            __syncwarp();
        }
    } else {
        regs_inc<kPaRegsSoftmax>();
        // ---- softmax: thread = row
        const int t = warp >> 2, r = tid & 127;
        const int ns = t ? nstep1 : nstep0;
        const int rt = r / a.gp, rg = r - rt * a.gp;
        const bool live = rt < job->n_tok[t] && seq >= 0;
        const int lim = live ? prompt_limit(a, seq, job->tok[t] + rt, job->lq, job->lk) : 0;
        const int clear = ns > 0 ? prompt_limit(a, seq, job->tok[t], job->lq, job->lk) : 0;   // fewest keys of the tile
        const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t tS = tmem + 128 * t + lane_base, tO = tmem + 256 + 128 * t + lane_base;
        const float c = a.scale_log2, slack = 8.0f / c;
        // fp16 weights carry 2^6 (at most 2^14, with m 2^8 behind): beside a key of weight 1 the others are good to 2^-31
        // of it. Without, to 2^-25: 16384 keys that share a 90th were off by 2 % of themselves, now by 2^-10.
        constexpr float kUp = kBf16 ? 0.f : 6.f;
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        // the ring is freed in pairs: K tile 0, then p: V tile p - 1 and K tile p. When the scores of step 2 p +
        // 1 are in, this tile's products with pair p are done.
        int freed = 0;
        for (int i = 0; i < ns; ++i) {
            const uint32_t tB = tS + kPaStep * (i & 1);
            ok = __all_sync(0xffffffffu, mbar_wait(s_full + 2 * t + (i & 1), (uint32_t)(i >> 1) & 1u)) != 0;
            if (!ok) break;
            tc_fence_after();
            if (i & 1) {
                if (r == 0) mbar_arrive(kv_empty + (freed & 3));
                ++freed;
            }
            uint32_t s[2][32];
            tmem_ld_32x32b_x32(tB, s[0]);
            tmem_ld_32x32b_x32(tB + 32, s[1]);
            tmem_ld_wait();
            tmem_ready(s[0]);
            tmem_ready(s[1]);
            const bool masked = (i + 1) * kPaStep > clear;
            const int left = lim - i * kPaStep;
            float mx[2];
            #pragma unroll
            for (int x = 0; x < 2; ++x) {
                if (masked) {
                    #pragma unroll
                    for (int y = 0; y < 32; ++y)
                        if (32 * x + y >= left) s[x][y] = 0xFF800000u;   // -inf
                }
                float a0 = __uint_as_float(s[x][0]), a1 = __uint_as_float(s[x][1]);
                #pragma unroll
                for (int y = 2; y < 32; y += 4) {
                    a0 = max_nan(a0, __uint_as_float(s[x][y]), __uint_as_float(s[x][y + 1]));
                    if (y + 2 < 32) a1 = max_nan(a1, __uint_as_float(s[x][y + 2]), __uint_as_float(s[x][y + 3]));
                }
                mx[x] = max_nan(a0, a1, a1);
            }
            const float top = max_nan(mx[0], mx[1], mx[1]);
            // a seen score that is NaN or +infinity: from here on the row's sum, and with it the row, is NaN
            if (!(top <= 3.402823466e38f)) l = __int_as_float(0x7fffffff);
            if (__any_sync(0xffffffffu, top - m > slack)) {   // m = -infinity: any finite top
                const float mn = fmaxf(m, top);
                if (i > 0) {
                    // rescale O once the products so far are in (this step's are not issued before its P is there)
                    ok = __all_sync(0xffffffffu, i + 1 < ns ? mbar_wait(s_full + 2 * t + ((i + 1) & 1), (uint32_t)((i + 1) >> 1) & 1u)
                                                            : mbar_wait(o_prev + t, 0)) != 0;
                    if (!ok) break;
                    tc_fence_after();
                    const float alpha = m == -INFINITY ? 0.f : ex2((m - mn) * c);
                    l *= alpha;
                    #pragma unroll 1
                    for (int x = 0; x < D / 16; ++x) {
                        uint32_t o[16];
                        tmem_ld_32x32b_x16(tO + 16 * x, o);
                        tmem_ld_wait();
                        tmem_ready(o);
                        #pragma unroll
                        for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * alpha);
                        tmem_st_32x32b_x16(tO + 16 * x, o);
                    }
                    tmem_st_wait();
                }
                m = mn;
            }
            const float mc = m == -INFINITY ? 0.f : kUp - m * c;
            const float2 c2 = make_float2(c, c), mc2 = make_float2(mc, mc);
            float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            uint32_t p[32];
            auto weights = [&](auto masked_tag) {
                #pragma unroll
                for (int x = 0; x < 32; ++x) {
                    const int e = 2 * x;
                    float2 v = fma2(make_float2(__uint_as_float(s[e >> 5][e & 31]), __uint_as_float(s[e >> 5][(e & 31) + 1])),
                                    c2, mc2);
                    // a masked weight has to be 0 exactly: those blocks take no polynomial
                    if (!decltype(masked_tag)::value && (x & 7) < kPoly) {
                        v = ex2_poly<!kBf16>(v);
                    } else {
                        v.x = ex2(v.x);
                        v.y = ex2(v.y);
                    }
                    sum[x & 1] = add2(sum[x & 1], v);
                    p[x] = pack2<T>(v.x, v.y);
                }
            };
            if (masked) weights(std::true_type{});
            else weights(std::false_type{});
            tmem_st_32x32b_x32(tB, p);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 2 * t + (i & 1));
            l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        }
        // ---- O / l
        if (ok && ns > 0) ok = mbar_wait(o_done + t, 0);
        ok = __all_sync(0xffffffffu, ok);
        // the rest of the ring's tiles, and those that only the other tile uses, once they are there
        if (ok && r == 0)
            for (; freed <= nblk && nblk > 0; ++freed) {
                const int first = max(2 * freed - 1, 0), last = min(2 * freed, 2 * nblk - 1);
                for (int x = first; x <= last && ok; ++x) ok = mbar_wait(kv_full + x % kStages, (uint32_t)(x / kStages) & 1u);
                if (!ok) break;
                mbar_arrive(kv_empty + (freed & 3));
            }
        ok = __all_sync(0xffffffffu, ok);
        if (ok) {
            tc_fence_after();
            // keys that all score -infinity leave no maximum: NaN, as 0 / 0 is
            const float inv = lim == 0 ? 0.f : m == -INFINITY ? __int_as_float(0x7fffffff) : 1.0f / l;
            // Through the tile of Q, which no product reads any more, each warp its own 32 rows, so that a
            // store writes whole rows (thread by thread, 16 bytes of 32 rows at a time, the stores took
            // longer than a block). Chunk c of a row lies at c ^ row.
            constexpr int kChunks = D / 8;
            uint4* stage = reinterpret_cast<uint4*>(sq + t * kTile) + (warp & 3) * 32 * kChunks;
            #pragma unroll 1
            for (int x = 0; x < D / 32; ++x) {
                uint32_t o[32];
                if (ns > 0) {
                    tmem_ld_32x32b_x32(tO + 32 * x, o);
                    tmem_ld_wait();
                    tmem_ready(o);
                }
                #pragma unroll
                for (int y = 0; y < 4; ++y) {
                    uint4 w = make_uint4(0u, 0u, 0u, 0u);
                    if (ns > 0 && lim > 0) {
                        w.x = pack2<T>(__uint_as_float(o[8 * y]) * inv, __uint_as_float(o[8 * y + 1]) * inv);
                        w.y = pack2<T>(__uint_as_float(o[8 * y + 2]) * inv, __uint_as_float(o[8 * y + 3]) * inv);
                        w.z = pack2<T>(__uint_as_float(o[8 * y + 4]) * inv, __uint_as_float(o[8 * y + 5]) * inv);
                        w.w = pack2<T>(__uint_as_float(o[8 * y + 6]) * inv, __uint_as_float(o[8 * y + 7]) * inv);
                    }
                    stage[lane * kChunks + ((4 * x + y) ^ (lane & (kChunks - 1)))] = w;
                }
            }
            __syncwarp();
            const long long to = live ? ((long long)(job->q0 + job->tok[t] + rt) * a.n_q + head0 + rg) * a.d : -1;
            constexpr int kRowsAtOnce = 32 / kChunks;
            const int ch = lane % kChunks;
            #pragma unroll 4
            for (int x = 0; x < 32; x += kRowsAtOnce) {
                const int row = x + lane / kChunks;
                const long long at = __shfl_sync(0xffffffffu, to, row);
                if (at >= 0 && 8 * ch < a.d)
                    *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + at + 8 * ch) = stage[row * kChunks + (ch ^ (row & (kChunks - 1)))];
            }
            __syncwarp();
            if (ns > 0 && *reinterpret_cast<volatile int*>(&job->bad[t])) {
                __syncwarp();
                for (int x = 0; x < 32; ++x) {
                    const int xr = __shfl_sync(0xffffffffu, rt, x), xg = __shfl_sync(0xffffffffu, rg, x);
                    const int xl = __shfl_sync(0xffffffffu, lim, x);
                    if (__shfl_sync(0xffffffffu, (int)live, x))
                        prompt_row<T>(a, job->q0 + job->tok[t] + xr, head0 + xg, job->k0, xl);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Tensor map of [tokens][heads][d] 16-bit elements: boxes of 64 channels (zeros
// past d) x box_heads x box_tok, rows of 128 bytes swizzled.
bool make_tmap_heads(CUtensorMap* map, const HeadsIn& h, int tokens, int heads, int d, int box_heads, int box_tok,
                     bool bf16) {
    auto fn = get_encode_fn();
    if (!fn || tokens <= 0) return false;
    // a stride that is never taken still has to be a legal one
    const long long head = heads > 1 ? h.head : d, tok = tokens > 1 ? h.tok : (long long)heads * head;
    if ((reinterpret_cast<uintptr_t>(h.p) & 15) || head <= 0 || tok <= 0 || head % 8 || tok % 8) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)head * 2, (cuuint64_t)tok * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tok};
    const cuuint32_t estr[3] = {1, 1, 1};
    return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(h.p),
              dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D>
cudaError_t prompt_launch(const PromptArgs& a, cudaStream_t st) {
    static std::atomic<unsigned long long> ready{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(ready.load() & bit)) {
        e = cudaFuncSetAttribute(prompt_tc_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)pa_smem(D));
        if (e != cudaSuccess) return e;
        // the split of the registers must not ask for more than the block is launched with
        cudaFuncAttributes fa;
        e = cudaFuncGetAttributes(&fa, prompt_tc_kernel<T, D>);
        if (e != cudaSuccess) return e;
        if (fa.numRegs < kPaRegsAtLaunch) return cudaErrorInvalidConfiguration;
        ready.fetch_or(bit);
    }
    CUtensorMap mq, mk, mv;
    constexpr bool bf16 = !std::is_same<T, __half>::value;
    if (!make_tmap_heads(&mq, a.q, a.total_q, a.n_q, a.d, a.gp, a.tile_tok, bf16)) return cudaErrorInvalidValue;
    if (a.total_k > 0) {
        if (!make_tmap_heads(&mk, a.k, a.total_k, a.n_kv, a.d, 1, kPaKeys, bf16) ||
            !make_tmap_heads(&mv, a.v, a.total_k, a.n_kv, a.d, 1, kPaKeys, bf16))
            return cudaErrorInvalidValue;
    } else {
        mk = mv = mq;   // no key is loaded
    }
    // a sequence's last pair may be short: at most one more pair each than the tokens fill
    const long long pairs = (a.total_q + 2ll * a.tile_tok - 1) / (2 * a.tile_tok) + a.n_seq;
    const long long grid = pairs * (a.n_q / a.gp);
    if (grid > INT_MAX) return cudaErrorInvalidValue;
    return launch_k(prompt_tc_kernel<T, D>, dim3((unsigned)grid), dim3(kPaThreads), pa_smem(D), st, a, mq, mk, mv);
}

}  // namespace

cudaError_t prompt_attention(void* out, const HeadsIn& q, const HeadsIn& k, const HeadsIn& v, int type,
                             const int* cu_q, const int* cu_k, const int* prefix, int n_seq, int total_q, int total_k,
                             int n_q, int n_kv, int d, float scale, int causal, cudaStream_t st) {
    if (total_q <= 0 || n_seq <= 0) return cudaSuccess;
    PromptArgs a{q, k, v, out, cu_q, cu_k, prefix, n_seq, total_q, total_k, n_q, n_kv, d, causal, scale < 0.f,
                 fabsf(scale) * 1.4426950408889634f, 1, kPaRows};
    if (a.scale_log2 < 1e-30f) a.scale_log2 = 1e-30f;   // scale 0: equal weights, but a masked score stays -inf
    // the whole group shares a tile where that fills at least 120 of its 128
    // rows, else the largest part of it that does (1 always does)
    const int group = n_q / n_kv;
    for (int g = 1; g <= group && g <= kPaRows; ++g)
        if (group % g == 0 && kPaRows / g * g >= 120) a.gp = g;
    a.tile_tok = kPaRows / a.gp;
    cudaError_t e;
    if (type == kBF16) e = d > 64 ? prompt_launch<__nv_bfloat16, 128>(a, st) : prompt_launch<__nv_bfloat16, 64>(a, st);
    else if (type == kF16) e = d > 64 ? prompt_launch<__half, 128>(a, st) : prompt_launch<__half, 64>(a, st);
    else return cudaErrorInvalidValue;
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace vsb

// Attention over packed prompts: grouped heads, causal or dense, sequences of
// different lengths one after another in one array.
#include "serve_ops.h"
#include "launch.cuh"
#include "sm100.cuh"

namespace vsb {

namespace {

struct PromptArgs {
    HeadsIn q, k, v;
    void* out;
    const int *cu_q, *cu_k, *prefix;
    int n_seq, total_q, total_k, n_q, n_kv, d, causal;
    float scale_log2;   // scale * log2(e)
};

// keys that query i of a sequence of lq queries and lk keys sees: [0, limit)
__device__ __forceinline__ int prompt_limit(const PromptArgs& a, int seq, int i, int lq, int lk) {
    int lim = a.causal ? min(max(i + 1 + lk - lq, 0), lk) : lk;
    if (a.prefix) lim = max(lim, min(a.prefix[seq], lk));
    return lim;
}

// One warp a row, one key at a time: the definition with an online softmax.
template <typename T>
__global__ void __launch_bounds__(128)
prompt_row_kernel(const __grid_constant__ PromptArgs a) {
    const int lane = threadIdx.x & 31, row = blockIdx.x * 4 + (threadIdx.x >> 5), head = blockIdx.y;
    pdl_trigger();
    pdl_wait();
    if (row >= a.total_q) return;
    int seq = 0;
    while (seq < a.n_seq && a.cu_q[seq + 1] <= row) ++seq;
    if (seq >= a.n_seq || row < a.cu_q[seq]) return;
    float o[4] = {}, q[4] = {}, m = -INFINITY, l = 0.f;
    {
        const int q0 = a.cu_q[seq], k0 = max(a.cu_k[seq], 0), k1 = min(a.cu_k[seq + 1], a.total_k);
        const int kvh = head / (a.n_q / a.n_kv);
        const int lim = prompt_limit(a, seq, row - q0, a.cu_q[seq + 1] - q0, max(k1 - k0, 0));
        const T* qp = static_cast<const T*>(a.q.p) + (long long)row * a.q.tok + (long long)head * a.q.head;
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
            s *= a.scale_log2;
            const float mn = fmaxf(m, s), alpha = ex2(m - mn), w = ex2(s - mn);
            m = mn;
            l = fmaf(l, alpha, w);
            #pragma unroll
            for (int x = 0; x < 4; ++x)
                if (lane + 32 * x < a.d) o[x] = fmaf(o[x], alpha, w * to_f(vp[lane + 32 * x]));
        }
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    T* out = static_cast<T*>(a.out) + ((long long)row * a.n_q + head) * a.d;
    #pragma unroll
    for (int x = 0; x < 4; ++x)
        if (lane + 32 * x < a.d) out[lane + 32 * x] = from_f<T>(o[x] * inv);
}

}  // namespace

cudaError_t prompt_attention(void* out, const HeadsIn& q, const HeadsIn& k, const HeadsIn& v, int type,
                             const int* cu_q, const int* cu_k, const int* prefix, int n_seq, int total_q, int total_k,
                             int n_q, int n_kv, int d, float scale, int causal, cudaStream_t st) {
    if (total_q <= 0) return cudaSuccess;
    const PromptArgs a{q, k, v, out, cu_q, cu_k, prefix, n_seq, total_q, total_k, n_q, n_kv, d, causal,
                       scale * 1.4426950408889634f};
    const dim3 grid((unsigned)((total_q + 3) / 4), (unsigned)n_q);
    const cudaError_t e = type == kBF16 ? launch_k(prompt_row_kernel<__nv_bfloat16>, grid, dim3(128), 0, st, a)
                          : type == kF16 ? launch_k(prompt_row_kernel<__half>, grid, dim3(128), 0, st, a)
                                         : cudaErrorInvalidValue;
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace vsb

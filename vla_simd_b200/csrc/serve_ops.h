// Serving operators of a prompted policy: head norms + multi-axis rotary
// positions, packed prompt attention, the paged 4-bit key / value cache and the
// attention that reads it (include/vla_simd_cuda.h states their definitions).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace vsb {

// element types of the C ABI (VLA_TYPE_*)
enum : int { kF32 = 0, kF16 = 1, kBF16 = 2 };

// A [tokens][heads][head_dim] operand: strides in elements, channels contiguous.
struct HeadsIn {
    const void* p = nullptr;
    long long tok = 0, head = 0;
};

constexpr int kMaxPairs = 128;   // rotated channel pairs of one head (head_dim <= 256)

struct RopeTable {
    double turns[kMaxPairs];       // frequency of pair i over 2 pi
    unsigned char axis[kMaxPairs]; // the position axis pair i turns with
};

cudaError_t qk_norm_rope(void* q_out, void* k_out, int out_type, const HeadsIn& q, const HeadsIn& k, int in_type,
                         const int* pos, const RopeTable& tab, int rot, const float* qw, const float* kw, float eps,
                         int tokens, int n_q, int n_kv, int d, cudaStream_t st);

cudaError_t prompt_attention(void* out, const HeadsIn& q, const HeadsIn& k, const HeadsIn& v, int type,
                             const int* cu_q, const int* cu_k, const int* prefix, int n_seq, int total_q, int total_k,
                             int n_q, int n_kv, int d, float scale, int causal, cudaStream_t st);

// ------------------------------------------------------------ 4-bit cache
constexpr int kKv4Group = 32;    // channels that share a scale and a minimum
constexpr int kKv4Block = 16;    // tokens of one block

struct Kv4Cache {
    uint8_t* p = nullptr;        // [n_pages][n_kv][page / 16][20 * d]
    long long n_pages = 0;
    int page = 0, n_kv = 0, d = 0;
};

cudaError_t kv4_append(const Kv4Cache& c, const HeadsIn& k, const HeadsIn& v, int type, const long long* slots,
                       int tokens, cudaStream_t st);
cudaError_t kv4_read(const Kv4Cache& c, void* k_out, void* v_out, int type, const long long* slots, int tokens,
                     cudaStream_t st);

struct Kv4AttArgs {
    void* out = nullptr;         // [batch][queries][n_q][d]
    const void* q = nullptr;
    long long q_seq = 0, q_tok = 0, q_head = 0;
    int type = kF32;
    Kv4Cache cache;
    const int* table = nullptr;  // [batch][table_ld]
    long long table_ld = 0;
    int max_pages = 0;
    const int* lens = nullptr;
    int batch = 0, queries = 0, n_q = 0;
    float scale = 0.f;
    int causal = 1;
    void* ws = nullptr;
    unsigned long long ws_bytes = 0;
};
unsigned long long kv4_attention_ws_bytes(int batch, int queries, int n_q, int n_kv, int d, long long max_len);
cudaError_t kv4_attention(const Kv4AttArgs& a, cudaStream_t st);

}  // namespace vsb

// Launch wrappers of the operators of a serving step that lie beside the model's own path: log probabilities
// (kernels_logprobs.cu), the 4-bit K / V cache (kernels_kv_q4.cu) and the attention of packed prompts (attn_prompts.cu).  All are
// asynchronous on `st`; arguments have been checked by the caller.
#pragma once
#include "dtypes.cuh"
#include "kernels.cuh"

namespace wick {

// The device-side waits of the two attentions, for the calling thread's launches: rounds of try_wait after which one gives up (a round on a phase that does
// not end takes 1.48 us, 2^18 of them 0.39 s), and, for tests, arrivals that a copy's barrier wants and nobody makes.
struct ServingWaits {
    uint32_t rounds = 1u << 18, missing = 0;
};
ServingWaits& serving_waits();
#ifdef __CUDACC__
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// Behind a wait that ran out: copies and matrix instructions that are under way end within this time.
__device__ __forceinline__ void settle() {
    unsigned long long t0, t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
    for (int i = 0; i < 1000; i++) {
        __nanosleep(1000);
        asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
        if (t - t0 > 100000) break;
    }
}
#endif

constexpr int LOGPROBS_MAX_TOP = 64;
cudaError_t launch_token_logprobs(cudaStream_t st, const void* logits, int dtype, size_t row_stride, int n, int vocab, const int32_t* tokens,
                                  int top_n, float* logprob, float* entropy, int32_t* top_ids, float* top_logprobs);

// The 4-bit cache: for every (slot, KV head) max_seq rows of head_dim / 32 Q4_0 blocks (wick/src/quant.rs:13-20), quants and f16
// scales in planes of their own, so that a head's rows are one contiguous stream.
struct KvQ4 {
    uint8_t* q[2];   // keys, values: [n_slots][n_kv][max_seq][head_dim / 2]
    __half* d[2];    //               [n_slots][n_kv][max_seq][head_dim / 32]
    int n_slots, n_kv, max_seq, head_dim;
    __host__ __device__ size_t row(int slot, int kvh, int pos) const { return ((size_t)slot * n_kv + kvh) * max_seq + pos; }
};
constexpr int KV_Q4_TILE = 64;  // max_seq is a multiple of it: a tile of rows never leaves its (slot, KV head)
constexpr int KV_Q4_MAX_HEAD = 128;
constexpr uint32_t KV_Q4_MAX_ROWS = 0x7FFFFF00u;  // of an append or a reading: a row's number, and the numbers up to the end of its block, are ints
cudaError_t launch_kv_append_q4(cudaStream_t st, const KvQ4& c, const void* k, size_t k_stride, const void* v, size_t v_stride, int dtype, int n,
                                const int32_t* slots, const int32_t* positions);
cudaError_t launch_kv_read_q4(cudaStream_t st, const KvQ4& c, int n, const int32_t* slots, const int32_t* positions, float* k, float* v);
size_t attention_q4_workspace(int head_dim);
cudaError_t launch_attention_q4(cudaStream_t st, const KvQ4& c, const void* q, size_t q_stride, int dtype, int n, int n_heads, const int32_t* slots,
                                const int32_t* lengths, void* out, int zero_rest, void* workspace);

// Packed prompts.  Rows of q / k / v are q_stride / k_stride / v_stride elements apart; starts (and key_starts, NULL: the same)
// hold n_seqs + 1 offsets.
struct Prompts {
    const void *q, *k, *v;
    size_t q_stride, k_stride, v_stride;
    int dtype;
    const int32_t *starts, *key_starts;
    int n_seqs, n_tokens, n_keys, n_heads, n_kv, head_dim;
    void* out;
    int zero_rest;  // rows of out that belong to no sequence: set to zero (else left alone)
};
size_t attention_prompts_workspace(const Prompts& p);
cudaError_t launch_attention_prompts(cudaStream_t st, const Prompts& p, void* workspace);

}  // namespace wick

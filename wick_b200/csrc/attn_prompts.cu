// Causal attention of packed prompts with grouped heads: token j of a sequence with nq tokens and nk >= nq keys attends the keys
// t <= j + nk - nq of its own sequence; a token that has none (nk < nq - j) gets zeros.
#include "serving.cuh"

namespace wick {

namespace {

constexpr int PR_THREADS = 128, PR_MAX_HEAD = 128;

// One CTA per (token, query head): runs of 128 keys, a running maximum and sum.
template <class T>
__global__ void __launch_bounds__(PR_THREADS) k_attention_prompts(Prompts a) {
    __shared__ float qs[PR_MAX_HEAD], p[PR_THREADS], red[4];
    const int h = blockIdx.x, tid = threadIdx.x, hd = a.head_dim, kvh = h / (a.n_heads / a.n_kv);
    const long long token = blockIdx.y + (long long)blockIdx.z * 65535;
    if (token >= a.n_tokens) return;
    int seq = 0;
    while (seq < a.n_seqs && a.starts[seq + 1] <= token) seq++;
    if (seq == a.n_seqs || token < a.starts[seq]) return;  // a row of no sequence
    const int32_t* ks = a.key_starts ? a.key_starts : a.starts;
    const int k0 = max(0, min(ks[seq], a.n_keys)), nk = max(0, min(ks[seq + 1], a.n_keys) - k0);
    const int nq = a.starts[seq + 1] - a.starts[seq], j = (int)token - a.starts[seq];
    const int len = max(0, min(nk, j + 1 + nk - nq));
    const T* k = (const T*)a.k + (size_t)k0 * a.k_stride + kvh * hd;
    const T* v = (const T*)a.v + (size_t)k0 * a.v_stride + kvh * hd;
    const float scale = __fdiv_rn(1.0f, sqrtf((float)hd));
    if (tid < hd) qs[tid] = __fmul_rn(to_f32(((const T*)a.q)[(size_t)token * a.q_stride + h * hd + tid]), scale);
    float m = __int_as_float(0xFF800000), l = 0.0f, acc = 0.0f;
    for (int t0 = 0; t0 < len; t0 += PR_THREADS) {
        const int t = t0 + tid, nt = min(PR_THREADS, len - t0);
        __syncthreads();
        float s = __int_as_float(0xFF800000);
        if (t < len) {
            s = 0.0f;
            for (int d = 0; d < hd; d++) s = fmaf(qs[d], to_f32(k[(size_t)t * a.k_stride + d]), s);
        }
        float top = s;
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if ((tid & 31) == 0) red[tid >> 5] = top;
        __syncthreads();
        const float m2 = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        const float f = expf(m - m2);
        p[tid] = t < len ? expf(s - m2) : 0.0f;
        m = m2;
        __syncthreads();
        l *= f, acc *= f;
        for (int i = 0; i < nt; i++) {
            l += p[i];
            if (tid < hd) acc = fmaf(p[i], to_f32(v[(size_t)(t0 + i) * a.v_stride + tid]), acc);
        }
    }
    if (tid < hd) ((T*)a.out)[((size_t)token * a.n_heads + h) * hd + tid] = from_f32<T>(len ? acc / l : 0.0f);
}

}  // namespace

size_t attention_prompts_workspace(const Prompts&) { return 0; }

cudaError_t launch_attention_prompts(cudaStream_t st, const Prompts& a, void*) {
    const dim3 grid((unsigned)a.n_heads, (unsigned)(a.n_tokens < 65535 ? a.n_tokens : 65535), (unsigned)((a.n_tokens + 65534) / 65535));
    g_kernel_launches++;
    if (a.dtype == DT_F32)
        k_attention_prompts<float><<<grid, PR_THREADS, 0, st>>>(a);
    else if (a.dtype == DT_F16)
        k_attention_prompts<__half><<<grid, PR_THREADS, 0, st>>>(a);
    else
        k_attention_prompts<__nv_bfloat16><<<grid, PR_THREADS, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace wick

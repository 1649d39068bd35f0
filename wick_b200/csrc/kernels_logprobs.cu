// Log probabilities of given tokens, with the entropy and the largest alternatives, over rows of logits x:
//     m = max x,  S = sum exp(x - m),  T = sum exp(x - m) (x - m)
//     log p(t) = (x_t - m) - log S,    H = -sum p log p = log S - T / S
// One pass: every thread keeps a running (m, S, T) of its elements and rescales it when its maximum grows (S' = S e,
// T' = (T + S (m - m')) e with e = exp(m - m')); threads, then the CTAs of a row, are joined by the same rule.
//
// A cluster of 1 to 8 CTAs takes a row: as many as give every SM work (the rule in launch_token_logprobs), joined through
// distributed shared memory, so that the call is one launch and needs no workspace.  Bound: the read of the logits.
//
// Alternatives: the top_n-th largest of the threads' maxima is a bound that top_n elements reach and few others do.  A second read
// (the row is in L2 by then) collects what reaches it; candidates are ordered by counting, CTAs' lists are joined the same way.
// Where ties make too many candidates (a vocabulary that is masked but for a few tokens), top_n rounds of "largest key below the
// last one" follow instead.
//
// Sums: f32 within a thread's few hundred elements, f64 from there on (log S and T / S cancel for sharp rows).
// NaN counts as -inf, as for the argmax (wick/src/sampler.rs:8-19); logits are held to +-1e30, so that +inf and -inf need no case of
// their own: several +inf share the row, -inf has probability 0, a row of -inf alone has no probabilities (-inf, entropy 0).
#include <cooperative_groups.h>

#include "serving.cuh"

namespace wick {

namespace {

namespace cg = cooperative_groups;

constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32;
constexpr int LP_CAND = 1024;      // candidates that are ordered by counting
constexpr int LP_MAX_CLUSTER = 8;  // the portable limit
constexpr float LP_BOUND = 1e30f;  // (a thousand of them still add up to a finite number)

__device__ __forceinline__ float held(float x) { return fminf(fmaxf(x, -LP_BOUND), LP_BOUND); }  // (NaN: the lower bound)
// Descending order of (value, ascending index) as descending whole numbers; -0 equals +0.
__device__ __forceinline__ uint32_t value_key(float x) {
    const uint32_t b = __float_as_uint(__fadd_rn(x, 0.0f));
    return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }
__device__ __forceinline__ unsigned long long full_key(float x, uint32_t i) { return ((unsigned long long)value_key(x) << 32) | (0xFFFFFFFFu - i); }

struct Running {
    float m, s, t;
    template <int N>
    __device__ __forceinline__ void add(const float (&x)[N]) {
        float top = m;
#pragma unroll
        for (int i = 0; i < N; i++) top = fmaxf(top, x[i]);
        if (top > m) {
            const float d = __fsub_rn(m, top), e = expf(d);
            t = __fmul_rn(fmaf(s, d, t), e);
            s = __fmul_rn(s, e);
            m = top;
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float d = __fsub_rn(x[i], m), e = expf(d);
            s = __fadd_rn(s, e);
            t = fmaf(e, d, t);
        }
    }
};
struct Joined {
    double s, t;
    float m;
    __device__ __forceinline__ void join(float m2, double s2, double t2) {
        const float top = fmaxf(m, m2);
        const double d1 = (double)m - top, d2 = (double)m2 - top;
        const double e1 = d1 == 0.0 ? 1.0 : (double)expf((float)d1), e2 = d2 == 0.0 ? 1.0 : (double)expf((float)d2);
        t = (s > 0.0 ? (t + s * d1) * e1 : 0.0) + (s2 > 0.0 ? (t2 + s2 * d2) * e2 : 0.0);
        s = s * e1 + s2 * e2;
        m = top;
    }
};

template <class T>
struct Slice {  // the part of a row that a CTA reads: 16-byte pieces [v0, v1), and single elements before and behind the row's aligned body
    const T* row;
    int head, n_vec, v0, v1, tail0, tail1, head1;
    static constexpr int V = 16 / sizeof(T);
    __device__ __forceinline__ Slice(const T* p, int vocab, int rank, int ctas) : row(p) {
        head = min(vocab, (int)(((16 - ((uintptr_t)p & 15)) & 15) / sizeof(T)));
        n_vec = (vocab - head) / V;
        v0 = (int)((long long)n_vec * rank / ctas), v1 = (int)((long long)n_vec * (rank + 1) / ctas);
        head1 = rank == 0 ? head : 0;
        tail0 = head + n_vec * V, tail1 = rank == ctas - 1 ? vocab : tail0;
    }
    __device__ __forceinline__ int index(int vec) const { return head + vec * V; }
    __device__ __forceinline__ void load(int vec, float (&x)[V]) const {
        unpack16(__ldg(reinterpret_cast<const uint4*>(row + head) + vec), x, (const T*)nullptr);
#pragma unroll
        for (int i = 0; i < V; i++) x[i] = held(x[i]);
    }
    // The at most one single element of this thread (a head or tail is shorter than 16 elements): its index or -1.
    __device__ __forceinline__ int single() const {
        const int i = threadIdx.x;
        if (i < head1) return i;
        return i - head1 < tail1 - tail0 ? tail0 + i - head1 : -1;
    }
    __device__ __forceinline__ float at(int i) const { return held(to_f32(row[i])); }
};

template <class T>
__global__ void __launch_bounds__(LP_THREADS) k_token_logprobs(const T* __restrict__ logits, size_t row_stride, int vocab,
                                                               const int32_t* __restrict__ tokens, int top_n, float* __restrict__ logprob,
                                                               float* __restrict__ entropy, int32_t* __restrict__ top_ids,
                                                               float* __restrict__ top_logprobs) {
    pdl_enter(logits, tokens, logprob, entropy, top_ids, top_logprobs);
    __shared__ double sh_s[LP_WARPS], sh_t[LP_WARPS];
    __shared__ float sh_m[LP_WARPS];
    __shared__ Joined part;                              // the CTA's, read by the row's first CTA
    __shared__ unsigned long long best[LOGPROBS_MAX_TOP];  // the CTA's top_n keys, descending
    __shared__ unsigned long long cand[LP_CAND];
    __shared__ uint32_t sh_key[LP_THREADS];
    __shared__ int n_cand;
    __shared__ uint32_t sh_floor;
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), row = blockIdx.x / ctas;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Slice<T> sl(logits + (size_t)row * row_stride, vocab, rank, ctas);
    constexpr int V = Slice<T>::V;

    Running r{-LP_BOUND, 0.0f, 0.0f};
    const int one = sl.single();
    if (one >= 0) {
        const float x[1] = {sl.at(one)};
        r.add(x);
    }
    int v = sl.v0 + tid;
    for (; v + 3 * LP_THREADS < sl.v1; v += 4 * LP_THREADS) {
        float x[4][V];
#pragma unroll
        for (int u = 0; u < 4; u++) sl.load(v + u * LP_THREADS, x[u]);
#pragma unroll
        for (int u = 0; u < 4; u++) r.add(x[u]);
    }
    for (; v < sl.v1; v += LP_THREADS) {
        float x[V];
        sl.load(v, x);
        r.add(x);
    }
    const float thread_max = r.m;
    Joined j{(double)r.s, (double)r.t, r.m};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, j.m, o);
        const double s2 = __shfl_xor_sync(0xffffffffu, j.s, o), t2 = __shfl_xor_sync(0xffffffffu, j.t, o);
        j.join(m2, s2, t2);
    }
    if (lane == 0) sh_m[warp] = j.m, sh_s[warp] = j.s, sh_t[warp] = j.t;
    if (tid == 0) n_cand = 0;
    sh_key[tid] = value_key(thread_max);
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < LP_WARPS; w++) j.join(sh_m[w], sh_s[w], sh_t[w]);
        part = j;
    }

    if (top_n > 0) {
        // the top_n-th largest of the threads' maxima, equal ones in thread order
        const uint32_t mine = sh_key[tid];
        int above = 0;
        for (int i = 0; i < LP_THREADS; i++) above += sh_key[i] > mine || (sh_key[i] == mine && i < tid);
        if (above == top_n - 1) sh_floor = mine;
        if (tid < top_n) best[tid] = 0;
        __syncthreads();
        const uint32_t floor_key = sh_floor;
        auto offer = [&](float x, int i) {
            if (value_key(x) >= floor_key) {
                const int at = atomicAdd(&n_cand, 1);
                if (at < LP_CAND) cand[at] = full_key(x, (uint32_t)i);
            }
        };
        if (mine >= floor_key) {  // (threads whose maximum lies below have nothing to offer)
            if (one >= 0) offer(sl.at(one), one);
            for (int u = sl.v0 + tid; u < sl.v1; u += LP_THREADS) {
                float x[V];
                sl.load(u, x);
#pragma unroll
                for (int i = 0; i < V; i++) offer(x[i], sl.index(u) + i);
            }
        }
        __syncthreads();
        const int n = n_cand;
        if (n <= LP_CAND) {
            for (int c = tid; c < n; c += LP_THREADS) {
                const unsigned long long k = cand[c];
                int p = 0;
                for (int i = 0; i < n; i++) p += cand[i] > k;
                if (p < top_n) best[p] = k;
            }
        } else {
            unsigned long long last = ~0ull;
            for (int p = 0; p < top_n; p++) {
                unsigned long long top = 0;
                auto look = [&](float x, int i) {
                    const unsigned long long k = full_key(x, (uint32_t)i);
                    if (k < last && k > top) top = k;
                };
                if (one >= 0) look(sl.at(one), one);
                for (int u = sl.v0 + tid; u < sl.v1; u += LP_THREADS) {
                    float x[V];
                    sl.load(u, x);
#pragma unroll
                    for (int i = 0; i < V; i++) look(x[i], sl.index(u) + i);
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                __syncthreads();
                if (lane == 0) cand[warp] = top;
                __syncthreads();
                for (int w = 0; w < LP_WARPS; w++) top = max(top, cand[w]);
                last = top;
                if (tid == 0) best[p] = top;
            }
        }
    }
    __syncthreads();
    if (ctas > 1) cluster.sync();
    if (rank == 0) {
        if (tid == 0) {
            for (int c = 1; c < ctas; c++) {
                const Joined* o = cluster.map_shared_rank(&part, c);
                part.join(o->m, o->s, o->t);
            }
        }
        if (top_n > 0 && ctas > 1) {
            // lists of keys that differ from one another: the place in the whole is the number of larger ones
            for (int c = tid; c < ctas * top_n; c += LP_THREADS) cand[c] = cluster.map_shared_rank(best, c / top_n)[c % top_n];
        }
        __syncthreads();
        const bool none = part.m <= -LP_BOUND;
        const double lse = log(part.s);
        const float ninf = __int_as_float(0xFF800000);
        auto log_p = [&](float x) {  // (beside a +inf, everything finite has probability 0)
            const float p = (float)((double)x - (double)part.m - lse);
            return none || x <= -LP_BOUND || p <= -0.5f * LP_BOUND ? ninf : p;
        };
        if (tid == 0) {
            const int t = tokens[row];
            logprob[row] = t >= 0 && t < vocab ? log_p(sl.at(t)) : ninf;
            entropy[row] = none ? 0.0f : (float)(lse - part.t / part.s);
        }
        if (top_n > 0) {
            const int total = ctas > 1 ? ctas * top_n : top_n;
            const unsigned long long* keys = ctas > 1 ? cand : best;
            for (int c = tid; c < total; c += LP_THREADS) {
                const unsigned long long k = keys[c];
                int p = 0;
                for (int i = 0; i < total; i++) p += keys[i] > k;
                if (k != 0 && p < top_n) {
                    top_ids[(size_t)row * top_n + p] = (int32_t)(0xFFFFFFFFu - (uint32_t)k);
                    top_logprobs[(size_t)row * top_n + p] = log_p(key_value((uint32_t)(k >> 32)));
                }
            }
        }
    }
    if (ctas > 1) cluster.sync();  // the first CTA has read the others' shared memory
}

template <class T>
cudaError_t launch_typed(cudaStream_t st, const void* logits, size_t row_stride, int n, int vocab, const int32_t* tokens, int top_n, float* logprob,
                         float* entropy, int32_t* top_ids, float* top_logprobs) {
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if ((e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return e;
    // CTAs to a row: doubled while every SM would still have at most four of them and each at least two rounds of loads.
    int ctas = 1;
    while (ctas < LP_MAX_CLUSTER && (long long)n * ctas * 2 <= 4ll * sms && vocab / (ctas * 2) >= 2 * LP_THREADS * (16 / (int)sizeof(T))) ctas *= 2;
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)ctas, attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)n * (unsigned)ctas);
    cfg.blockDim = dim3(LP_THREADS);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    g_kernel_launches++;
    return cudaLaunchKernelEx(&cfg, k_token_logprobs<T>, static_cast<const T*>(logits), row_stride, vocab, tokens, top_n, logprob, entropy, top_ids,
                              top_logprobs);
}

}  // namespace

cudaError_t launch_token_logprobs(cudaStream_t st, const void* logits, int dtype, size_t row_stride, int n, int vocab, const int32_t* tokens,
                                  int top_n, float* logprob, float* entropy, int32_t* top_ids, float* top_logprobs) {
    auto* launch = dtype == DT_F32 ? launch_typed<float> : dtype == DT_F16 ? launch_typed<__half> : launch_typed<__nv_bfloat16>;
    return launch(st, logits, row_stride, n, vocab, tokens, top_n, logprob, entropy, top_ids, top_logprobs);
}

}  // namespace wick

// Log probabilities of given tokens, with the entropy and the largest alternatives, over rows of logits x:
//     m = max x,  S = sum exp(x - m),  T = sum exp(x - m) (x - m)
//     log p(t) = (x_t - m) - log S,    H = -sum p log p = log S - T / S
// One pass: every thread keeps a running (m, S, T) of its elements, 32 at a time, and rescales it when its maximum grows (S' = S e,
// T' = (T + S (m - m')) e with e = exp(m - m')); threads, then the CTAs of a row, are joined by the same rule.
//
// A cluster of 1 to 8 CTAs takes a row: as many as give every SM work (the rule in launch_token_logprobs), joined through
// distributed shared memory, so that the call is one launch and needs no workspace.
//
// Alternatives: from the threads' maxima follows a value that top_n elements reach and few others do.  What reaches it is collected, from
// registers where the CTA's part of the row fits them and by a second read otherwise (L2 has it by then); candidates are ordered by counting, the
// CTAs' lists are joined the same way.
// Where ties make too many candidates (a vocabulary that is masked but for a few tokens), top_n rounds of "largest key below the
// last one" follow instead.
//
// On a B200: 2500 rows of 50021 in bf16 57 us (4.4 TB/s, 67 % of a copy's rate; special function unit 58 %, issue slots 52 %: a thread's loads and its
// arithmetic alternate), 64 rows of 65536 in f32 with twenty alternatives 14 us, one with five 7 us (the cluster's barriers and the candidates, one step
// after the other).
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

constexpr float LOG2E = 1.44269504088896341f;
__device__ __forceinline__ float max_nan(float a, float b, float c) {  // (NaN if one is)
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float min_nan(float a, float b, float c) {
    float r;
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// A thread's running maximum and sums, and one step of them by N values: half an instruction each for the maximum, the minimum, the difference,
// its product with log2 e and the two sums, one for the exponential.
struct Running {
    float m = -LP_BOUND;
    f32x2 s = 0, t = 0;  // (two zeros)
    template <int N>
    __device__ __forceinline__ float add(float (&x)[N]) {  // the largest of them
        static_assert(N == 1 || N % 2 == 0, "pairs");
        float top = x[0], low = x[0];
#pragma unroll
        for (int i = 1; i + 1 < N; i += 2) top = max_nan(top, x[i], x[i + 1]), low = min_nan(low, x[i], x[i + 1]);
        if (N % 2 == 0) top = max_nan(top, top, x[N - 1]), low = min_nan(low, low, x[N - 1]);
        if (!(top <= LP_BOUND && low >= -LP_BOUND)) {  // infinities, NaN
            top = -LP_BOUND;
#pragma unroll
            for (int i = 0; i < N; i++) x[i] = held(x[i]), top = fmaxf(top, x[i]);
        }
        if (top > m) {
            const float d = __fsub_rn(m, top), e = exp2_approx(__fmul_rn(d, LOG2E));
            t = mul2(fma2(s, pack2(d, d), t), pack2(e, e));
            s = mul2(s, pack2(e, e));
            m = top;
        }
        if constexpr (N == 1) {
            const float d = __fsub_rn(x[0], m), e = exp2_approx(__fmul_rn(d, LOG2E));
            s = add2(s, pack2(e, 0.0f));
            t = add2(t, pack2(__fmul_rn(e, d), 0.0f));
        } else {
            const f32x2 minus = pack2(-m, -m), log2e = pack2(LOG2E, LOG2E);
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                const f32x2 d = add2(pack2(x[i], x[i + 1]), minus);
                float y0, y1;
                unpack2(mul2(d, log2e), y0, y1);
                const f32x2 e = pack2(exp2_approx(y0), exp2_approx(y1));
                s = add2(s, e);
                t = fma2(e, d, t);
            }
        }
        return top;
    }
};
struct Joined {
    double s, t;
    float m;
    // The join of the 32 lanes' sums, in a fixed order, in every lane.
    __device__ __forceinline__ void over_lanes() {
        float top = m;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const double d = (double)m - (double)top, f = m == top ? 1.0 : (double)exp2_approx(__fmul_rn(__fsub_rn(m, top), LOG2E));
        t = s > 0.0 ? (t + s * d) * f : 0.0;
        s *= f;
        m = top;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o), t += __shfl_xor_sync(0xffffffffu, t, o);
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
    }
    // The at most one single element of this thread (a head or tail is shorter than 16 elements): its index or -1.
    __device__ __forceinline__ int single() const {
        const int i = threadIdx.x;
        if (i < head1) return i;
        return i - head1 < tail1 - tail0 ? tail0 + i - head1 : -1;
    }
    __device__ __forceinline__ float at(int i) const { return to_f32(row[i]); }
};

// HELD: the CTA's part of the row stays in registers (at most LP_HELD elements per thread), and is not read a second time for the alternatives.
// Otherwise the largest of every 32 elements is noted (of the first LP_CHUNKS of a thread), and only those that can hold an alternative are.
constexpr int LP_HELD = 32, LP_CHUNKS = 24;
template <class T, bool HELD>
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
    __shared__ int n_cand;
    __shared__ uint32_t sh_floor[LP_WARPS];
    __shared__ float chunk_max[HELD ? 1 : LP_CHUNKS][LP_THREADS];
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), row = blockIdx.x / ctas;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Slice<T> sl(logits + (size_t)row * row_stride, vocab, rank, ctas);
    constexpr int V = Slice<T>::V, AT_ONCE = LP_HELD / V;  // elements of a load; loads that are under way together

    Running r;
    const int one = sl.single();
    float x_one[1] = {-LP_BOUND};
    if (one >= 0) {
        x_one[0] = sl.at(one);
        r.add(x_one);
    }
    float x[LP_HELD];
    if constexpr (HELD) {
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) {
            const int v = sl.v0 + tid + u * LP_THREADS;
            float y[V];
#pragma unroll
            for (int i = 0; i < V; i++) y[i] = -LP_BOUND;
            if (v < sl.v1) sl.load(v, y);
#pragma unroll
            for (int i = 0; i < V; i++) x[u * V + i] = y[i];
        }
        r.add(x);
    } else {
        int v = sl.v0 + tid, chunk = 0;
        for (; v + (AT_ONCE - 1) * LP_THREADS < sl.v1; v += AT_ONCE * LP_THREADS) {
#pragma unroll
            for (int u = 0; u < AT_ONCE; u++) {
                float y[V];
                sl.load(v + u * LP_THREADS, y);
#pragma unroll
                for (int i = 0; i < V; i++) x[u * V + i] = y[i];
            }
            const float top = r.add(x);
            if (chunk < LP_CHUNKS) chunk_max[HELD ? 0 : chunk][tid] = top;
            chunk++;
        }
        float top = -LP_BOUND;
        for (; v < sl.v1; v += LP_THREADS) {
            float y[V];
            sl.load(v, y);
            top = fmaxf(top, r.add(y));
        }
        if (chunk < LP_CHUNKS) chunk_max[HELD ? 0 : chunk][tid] = top;
    }
    const uint32_t mine = value_key(r.m);
    Joined j;
    {
        float s0, s1, t0, t1;
        unpack2(r.s, s0, s1);
        unpack2(r.t, t0, t1);
        j.s = (double)s0 + s1, j.t = (double)t0 + t1, j.m = r.m;
    }
    j.over_lanes();
    if (lane == 0) sh_m[warp] = j.m, sh_s[warp] = j.s, sh_t[warp] = j.t;
    if (tid == 0) n_cand = 0;
    if (top_n > 0) {
        // A value that top_n elements of the CTA reach: each of A warps has k = top_n / A (upwards) threads whose maxima do, if it is the smallest
        // of those warps' k-th largest maxima.  (A: the warps whose threads all have elements.)
        const int full = max(1, min(LP_WARPS, (sl.v1 - sl.v0) / 32));
        // (A warp has 32 maxima.  Where that is too few, full is 1 and the row has fewer than 64 pieces: everything is a candidate.)
        uint32_t left = mine;
        uint32_t kth = value_key(-LP_BOUND);
        for (int k = 0; k < top_n && top_n <= 32 * full; k += full) {
            kth = __reduce_max_sync(0xffffffffu, left);
            const uint32_t at = __ballot_sync(0xffffffffu, left == kth);
            if (lane == __ffs(at) - 1) left = 0;
        }
        if (lane == 0) sh_floor[warp] = warp < full ? kth : 0xFFFFFFFFu;
    }
    __syncthreads();
    if (warp == 0) {
        j.m = lane < LP_WARPS ? sh_m[lane] : -LP_BOUND, j.s = lane < LP_WARPS ? sh_s[lane] : 0.0, j.t = lane < LP_WARPS ? sh_t[lane] : 0.0;
        j.over_lanes();
        if (lane == 0) part = j;
    }

    if (top_n > 0) {
        if (tid < top_n) best[tid] = 0;
        uint32_t floor_key = 0xFFFFFFFFu;
#pragma unroll
        for (int w = 0; w < LP_WARPS; w++) floor_key = min(floor_key, sh_floor[w]);
        const float floor_value = key_value(floor_key);
        auto offer = [&](float x, int i) {
            if (x >= floor_value) {
                const int at = atomicAdd(&n_cand, 1);
                if (at < LP_CAND) cand[at] = full_key(x, (uint32_t)i);
            }
        };
        if (mine >= floor_key) {  // (threads whose maximum lies below have nothing to offer)
            if (one >= 0) offer(held(x_one[0]), one);
            if constexpr (HELD) {
#pragma unroll
                for (int u = 0; u < AT_ONCE; u++) {
                    const int v = sl.v0 + tid + u * LP_THREADS;
                    if (v < sl.v1) {
#pragma unroll
                        for (int i = 0; i < V; i++) offer(x[u * V + i], sl.index(v) + i);
                    }
                }
            } else {
                int chunk = 0;
                for (int v = sl.v0 + tid; v < sl.v1; v += AT_ONCE * LP_THREADS, chunk++) {
                    if (chunk < LP_CHUNKS && !(chunk_max[HELD ? 0 : chunk][tid] >= floor_value)) continue;
                    float y[AT_ONCE][V];
#pragma unroll
                    for (int u = 0; u < AT_ONCE; u++) sl.load(min(v + u * LP_THREADS, sl.v1 - 1), y[u]);
#pragma unroll
                    for (int u = 0; u < AT_ONCE; u++)
                        if (v + u * LP_THREADS < sl.v1) {
#pragma unroll
                            for (int i = 0; i < V; i++) offer(held(y[u][i]), sl.index(v + u * LP_THREADS) + i);
                        }
                }
            }
        }
        __syncthreads();
        const int n = n_cand;
        if (n <= LP_CAND) {
            for (int c = tid; c < n; c += LP_THREADS) {
                const unsigned long long k = cand[c];
                int p = 0;
#pragma unroll 8
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
                if (one >= 0) look(held(x_one[0]), one);
                for (int u = sl.v0 + tid; u < sl.v1; u += LP_THREADS) {
                    float y[V];
                    sl.load(u, y);
#pragma unroll
                    for (int i = 0; i < V; i++) look(held(y[i]), sl.index(u) + i);
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
        if (ctas > 1 && warp == 0) {
            const Joined* o = cluster.map_shared_rank(&part, lane < ctas ? lane : 0);
            j.m = lane < ctas ? o->m : -LP_BOUND, j.s = lane < ctas ? o->s : 0.0, j.t = lane < ctas ? o->t : 0.0;
            j.over_lanes();
            __syncwarp();
            if (lane == 0) part = j;
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
            logprob[row] = t >= 0 && t < vocab ? log_p(held(sl.at(t))) : ninf;
            entropy[row] = none ? 0.0f : (float)(lse - part.t / part.s);
        }
        if (top_n > 0) {
            const int total = ctas > 1 ? ctas * top_n : top_n;
            const unsigned long long* keys = ctas > 1 ? cand : best;
            for (int c = tid; c < total; c += LP_THREADS) {
                const unsigned long long k = keys[c];
                int p = c % top_n;  // the larger ones of its own list, and of each other: lists descend
                if (total <= 64) {
                    p = 0;
#pragma unroll 8
                    for (int i = 0; i < total; i++) p += keys[i] > k;
                }
                for (int l = 0; total > 64 && l < total; l += top_n) {
                    if (l == c - c % top_n) continue;
                    int lo = 0, hi = top_n;
                    while (lo < hi) {
                        const int mid = (lo + hi) >> 1;
                        if (keys[l + mid] > k) lo = mid + 1;
                        else hi = mid;
                    }
                    p += lo;
                }
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
    const int loads = vocab / (16 / (int)sizeof(T));
    const bool held = (loads + ctas - 1) / ctas <= LP_HELD / (16 / (int)sizeof(T)) * LP_THREADS;
    return cudaLaunchKernelEx(&cfg, held ? k_token_logprobs<T, true> : k_token_logprobs<T, false>, static_cast<const T*>(logits), row_stride, vocab,
                              tokens, top_n, logprob, entropy, top_ids, top_logprobs);
}

}  // namespace

cudaError_t launch_token_logprobs(cudaStream_t st, const void* logits, int dtype, size_t row_stride, int n, int vocab, const int32_t* tokens,
                                  int top_n, float* logprob, float* entropy, int32_t* top_ids, float* top_logprobs) {
    auto* launch = dtype == DT_F32 ? launch_typed<float> : dtype == DT_F16 ? launch_typed<__half> : launch_typed<__nv_bfloat16>;
    return launch(st, logits, row_stride, n, vocab, tokens, top_n, logprob, entropy, top_ids, top_logprobs);
}

}  // namespace wick

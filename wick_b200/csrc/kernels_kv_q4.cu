// The 4-bit K / V cache: append (Q4_0 rounding) and read back; the attention over it is attn_q4.cu.
//
// A block is 32 values: d = m / -8 with m the value of largest magnitude (the first of equal ones), q = min(15, trunc(x / d + 8.5)) as
// x * (1 / d), d kept in f16; the value it stands for is f16(d) * (q - 8).  Byte i of a block's 16 holds value i in its low and value
// i + 16 in its high half (BlockQ4_0, wick/src/quant.rs:13-20, and the rounding of the files that carry it).
#include "serving.cuh"

namespace wick {

namespace {

constexpr int KV_THREADS = 256;

template <class T>
__device__ __forceinline__ float4 load4(const T* p, bool vec) {
    if (!vec) return make_float4(to_f32(p[0]), to_f32(p[1]), to_f32(p[2]), to_f32(p[3]));
    if constexpr (sizeof(T) == 4) {
        return *reinterpret_cast<const float4*>(p);
    } else {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        const T* h = reinterpret_cast<const T*>(&w);
        return make_float4(to_f32(h[0]), to_f32(h[1]), to_f32(h[2]), to_f32(h[3]));
    }
}

// Four values per lane, a block on 8 lanes; blocks of the keys first, then those of the values.  Bound: HBM at prompts (the rows once,
// 18 bytes per block out), the launch at a decode step's few rows.
template <class T>
__global__ void __launch_bounds__(KV_THREADS) k_kv_append_q4(KvQ4 c, const T* __restrict__ k, size_t k_stride, const T* __restrict__ v, size_t v_stride,
                                                             int n, const int32_t* __restrict__ slots, const int32_t* __restrict__ positions, int vec) {
    pdl_enter(k, v, slots, positions);
    const int per_head = c.head_dim / QK, per_row = c.n_kv * per_head;
    const size_t blocks = (size_t)n * per_row, t = (size_t)blockIdx.x * KV_THREADS + threadIdx.x;
    const size_t b = t / 8;
    const int e = (int)(t & 7);
    const bool real = b < 2 * blocks, val = b >= blocks;
    const size_t bb = real ? (val ? b - blocks : b) : 0;
    const int j = (int)(bb / per_row), in_row = (int)(bb % per_row);
    const int slot = slots[j], pos = positions[j];
    const bool keep = real && slot >= 0 && slot < c.n_slots && pos >= 0 && pos < c.max_seq;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (keep) x = load4((val ? v + (size_t)j * v_stride : k + (size_t)j * k_stride) + in_row * QK + 4 * e, vec != 0);
    // the first value of largest magnitude: within the lane, then over the block's lanes
    float m = x.x;
    if (fabsf(x.y) > fabsf(m)) m = x.y;
    if (fabsf(x.z) > fabsf(m)) m = x.z;
    if (fabsf(x.w) > fabsf(m)) m = x.w;
    int at = e;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o);
        const int at2 = __shfl_xor_sync(0xffffffffu, at, o);
        if (fabsf(m2) > fabsf(m) || (fabsf(m2) == fabsf(m) && at2 < at)) m = m2, at = at2;
    }
    const float d = __fdiv_rn(m, -8.0f), id = d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
    auto q4 = [id](float f) { return (uint32_t)fminf(fmaxf(truncf(__fadd_rn(__fmul_rn(f, id), 8.5f)), 0.0f), 15.0f); };
    const uint32_t w = q4(x.x) | q4(x.y) << 8 | q4(x.z) << 16 | q4(x.w) << 24;
    const uint32_t high = __shfl_down_sync(0xffffffffu, w, 4);
    if (!keep) return;
    const size_t row = c.row(slot, in_row / per_head, pos);
    const int blk = in_row % per_head;
    if (e < 4) *reinterpret_cast<uint32_t*>(c.q[val] + row * (c.head_dim / 2) + blk * 16 + 4 * e) = w | high << 4;
    if (e == 0) c.d[val][row * per_head + blk] = __float2half_rn(d);
}

// One thread per four bytes of quants: eight values.  A row that the cache does not have reads as zeros.
__global__ void __launch_bounds__(KV_THREADS) k_kv_read_q4(KvQ4 c, int n, const int32_t* __restrict__ slots, const int32_t* __restrict__ positions,
                                                           float* __restrict__ k, float* __restrict__ v) {
    pdl_enter(slots, positions, k, v);
    const int per_head = c.head_dim / QK, per_row = c.n_kv * per_head;
    const size_t words = (size_t)n * per_row * 4, t = (size_t)blockIdx.x * KV_THREADS + threadIdx.x;
    if (t >= 2 * words) return;
    const int val = t >= words;
    const size_t b = (val ? t - words : t) / 4;
    const int e = (int)(t & 3), j = (int)(b / per_row), in_row = (int)(b % per_row);
    const int slot = slots[j], pos = positions[j];
    float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
    if (slot >= 0 && slot < c.n_slots && pos >= 0 && pos < c.max_seq) {
        const size_t row = c.row(slot, in_row / per_head, pos);
        const uint32_t w = *reinterpret_cast<const uint32_t*>(c.q[val] + row * (c.head_dim / 2) + in_row % per_head * 16 + 4 * e);
        const float d = __half2float(c.d[val][row * per_head + in_row % per_head]);
        auto at = [&](int shift) { return __fmul_rn(d, (float)((int)((w >> shift) & 15u) - 8)); };
        lo = make_float4(at(0), at(8), at(16), at(24));
        hi = make_float4(at(4), at(12), at(20), at(28));
    }
    float* out = (val ? v : k) + b * QK + 4 * e;
    *reinterpret_cast<float4*>(out) = lo;
    *reinterpret_cast<float4*>(out + 16) = hi;
}

}  // namespace

cudaError_t launch_kv_append_q4(cudaStream_t st, const KvQ4& c, const void* k, size_t k_stride, const void* v, size_t v_stride, int dtype, int n,
                                const int32_t* slots, const int32_t* positions) {
    const size_t align = 4 * (size_t)dtype_bytes(dtype);
    const int vec = (((uintptr_t)k | (uintptr_t)v | k_stride * dtype_bytes(dtype) | v_stride * dtype_bytes(dtype)) & (align - 1)) == 0;
    const size_t threads = (size_t)n * c.n_kv * c.head_dim / 2;  // a quarter of each of the two rows
    const dim3 grid((unsigned)((threads + KV_THREADS - 1) / KV_THREADS)), block(KV_THREADS);
    g_kernel_launches++;
    if (dtype == DT_F32)
        return launch_pdl(st, k_kv_append_q4<float>, grid, block, 0, c, (const float*)k, k_stride, (const float*)v, v_stride, n, slots, positions, vec);
    if (dtype == DT_F16)
        return launch_pdl(st, k_kv_append_q4<__half>, grid, block, 0, c, (const __half*)k, k_stride, (const __half*)v, v_stride, n, slots, positions, vec);
    return launch_pdl(st, k_kv_append_q4<__nv_bfloat16>, grid, block, 0, c, (const __nv_bfloat16*)k, k_stride, (const __nv_bfloat16*)v, v_stride, n,
                      slots, positions, vec);
}

cudaError_t launch_kv_read_q4(cudaStream_t st, const KvQ4& c, int n, const int32_t* slots, const int32_t* positions, float* k, float* v) {
    const size_t threads = (size_t)n * c.n_kv * c.head_dim / 4;
    g_kernel_launches++;
    return launch_pdl(st, k_kv_read_q4, dim3((unsigned)((threads + KV_THREADS - 1) / KV_THREADS)), dim3(KV_THREADS), 0, c, n, slots, positions, k, v);
}

}  // namespace wick

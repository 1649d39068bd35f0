// The 4-bit K / V cache: append (Q4_0 rounding) and read back; the attention over it is attn_q4.cu.
//
// A block is 32 values: d = m / -8 with m the value of largest magnitude (the first of equal ones), q = min(15, trunc(x / d + 8.5)) as
// x * (1 / d), d kept in f16; the value it stands for is f16(d) * (q - 8).  Byte i of a block's 16 holds value i in its low and value
// i + 16 in its high half (BlockQ4_0, wick/src/quant.rs:13-20, and the rounding of the files that carry it).
#include "serving.cuh"

namespace wick {

namespace {

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

// Both kernels: a row (its keys, then its values) to threadIdx.y and, in turns, threadIdx.x; 8 threads to a block.  (One list of all blocks
// over the threads cost two divisions of 64-bit numbers each: 9 us for 4093 rows of 512 either way.)
constexpr int KV_THREADS = 256;
dim3 row_threads(const KvQ4& c, int per_block) {
    const int want = (2 * c.n_kv * (c.head_dim / QK) * per_block + 31) / 32 * 32, x = want < KV_THREADS ? want : KV_THREADS;  // (whole warps)
    return dim3((unsigned)x, (unsigned)(KV_THREADS / x));
}
// Rows that a thread has under way together: a row is two or three dependent trips to memory, and at prompts the SMs' threads are too few
// to hide them one by one; below, more blocks do.  (Rows of 512, one at a time / four, append: 512 rows 3.3 / 3.7 us, 1024 4.3 / 4.4, 2048 6.5 / 6.1, 4093 11.0 / 9.4;
// reading: 2.2 / 3.1, 3.0 / 3.3, 4.3 / 4.5, 6.8 / 6.6.  Rows of 1024 alike, rows of 64 gain from 4000 on: 0.7 us at most either way.)
constexpr int KV_MANY = 4, KV_MANY_FROM = 1024;

// Four values per lane, a block on 8 lanes.  4093 rows of 512 with their reading back: 15.4 us where the bytes take 5.8; it waits for memory (a row is two or
// three trips, a lane has 2 to 16 bytes of each) and on the blocks' arithmetic.  A decode step's few rows are bound by the launch (3.4 us both).
template <class T, int ROWS>
__global__ void __launch_bounds__(KV_THREADS) k_kv_append_q4(KvQ4 c, const T* __restrict__ k, size_t k_stride, const T* __restrict__ v, size_t v_stride,
                                                             int n, const int32_t* __restrict__ slots, const int32_t* __restrict__ positions, int vec) {
    pdl_enter(k, v, slots, positions);
    const int per_head = c.head_dim / QK, per_row = c.n_kv * per_head, j0 = blockIdx.x * ROWS * blockDim.y + threadIdx.y, e = threadIdx.x & 7;
    int slot[ROWS], pos[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
        const int j = j0 + r * blockDim.y;
        slot[r] = j < n ? slots[j] : -1, pos[r] = j < n ? positions[j] : -1;
    }
    const int turns = (16 * per_row + blockDim.x - 1) / blockDim.x;  // (as many for every lane of a warp: they exchange values)
    for (int turn = 0; turn < turns; turn++) {
        const int b = (turn * blockDim.x + threadIdx.x) >> 3;
        const bool val = b >= per_row, in = b < 2 * per_row;
        const int in_row = val ? b - per_row : b, head = in_row / per_head, blk = in_row - head * per_head;
        float4 x[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; r++) {  // (without asking whether the row is kept: one trip to memory less)
            const int j = j0 + r * blockDim.y;
            x[r] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (in && j < n) x[r] = load4((val ? v + (size_t)j * v_stride : k + (size_t)j * k_stride) + in_row * QK + 4 * e, vec != 0);
        }
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
            // the first value of largest magnitude: within the lane, then over the block's lanes
            float m = x[r].x;
            if (fabsf(x[r].y) > fabsf(m)) m = x[r].y;
            if (fabsf(x[r].z) > fabsf(m)) m = x[r].z;
            if (fabsf(x[r].w) > fabsf(m)) m = x[r].w;
            int at = e;
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) {
                const float m2 = __shfl_xor_sync(0xffffffffu, m, o);
                const int at2 = __shfl_xor_sync(0xffffffffu, at, o);
                if (fabsf(m2) > fabsf(m) || (fabsf(m2) == fabsf(m) && at2 < at)) m = m2, at = at2;
            }
            const float d = __fmul_rn(m, -0.125f), id = d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
            // x / d + 8.5 lies in [0.5, 16.5]: adding 2^23 downwards leaves its whole part in the lowest bits
            auto q4 = [id](float f) { return __float_as_uint(__fadd_rd(fminf(__fadd_rn(__fmul_rn(f, id), 8.5f), 15.5f), 8388608.0f)) & 15u; };
            const uint32_t w = q4(x[r].x) | q4(x[r].y) << 8 | q4(x[r].z) << 16 | q4(x[r].w) << 24;
            const uint32_t high = __shfl_down_sync(0xffffffffu, w, 4);
            if (!in || slot[r] < 0 || slot[r] >= c.n_slots || pos[r] < 0 || pos[r] >= c.max_seq) continue;
            const size_t row = c.row(slot[r], head, pos[r]);
            if (e < 4) *reinterpret_cast<uint32_t*>(c.q[val] + row * (c.head_dim / 2) + blk * 16 + 4 * e) = w | high << 4;
            if (e == 0) c.d[val][row * per_head + blk] = __float2half_rn(d);
        }
    }
}

// Four bytes of quants, eight values, per thread.  A row that the cache does not have reads as zeros.
template <int ROWS>
__global__ void __launch_bounds__(KV_THREADS) k_kv_read_q4(KvQ4 c, int n, const int32_t* __restrict__ slots, const int32_t* __restrict__ positions,
                                                           float* __restrict__ k, float* __restrict__ v) {
    pdl_enter(slots, positions, k, v);
    const int per_head = c.head_dim / QK, per_row = c.n_kv * per_head, j0 = blockIdx.x * ROWS * blockDim.y + threadIdx.y, e = threadIdx.x & 3;
    int slot[ROWS], pos[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
        const int j = j0 + r * blockDim.y;
        slot[r] = j < n ? slots[j] : -1, pos[r] = j < n ? positions[j] : -1;
    }
    for (int b = threadIdx.x >> 2; b < 2 * per_row; b += blockDim.x >> 2) {
        const bool val = b >= per_row;
        const int in_row = val ? b - per_row : b, head = in_row / per_head, blk = in_row - head * per_head;
        uint32_t w[ROWS];
        float d[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
            w[r] = 0, d[r] = 0.0f;
            if (slot[r] >= 0 && slot[r] < c.n_slots && pos[r] >= 0 && pos[r] < c.max_seq) {
                const size_t row = c.row(slot[r], head, pos[r]);
                w[r] = *reinterpret_cast<const uint32_t*>(c.q[val] + row * (c.head_dim / 2) + blk * 16 + 4 * e);
                d[r] = __half2float(c.d[val][row * per_head + blk]);
            } else {
                w[r] = 0x88888888u;  // (zeros without a sign)
            }
        }
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
            const int j = j0 + r * blockDim.y;
            if (j >= n) continue;
            auto at = [&](int shift) { return __fmul_rn(d[r], (float)((int)((w[r] >> shift) & 15u) - 8)); };
            float* out = (val ? v : k) + ((size_t)j * per_row + in_row) * QK + 4 * e;
            *reinterpret_cast<float4*>(out) = make_float4(at(0), at(8), at(16), at(24));
            *reinterpret_cast<float4*>(out + 16) = make_float4(at(4), at(12), at(20), at(28));
        }
    }
}

template <class T>
cudaError_t launch_append(cudaStream_t st, const KvQ4& c, const void* k, size_t k_stride, const void* v, size_t v_stride, int n, const int32_t* slots,
                          const int32_t* positions, int vec) {
    const dim3 block = row_threads(c, 8);
    const unsigned rows = n >= KV_MANY_FROM ? KV_MANY * block.y : block.y;
    g_kernel_launches++;
    return launch_pdl(st, n >= KV_MANY_FROM ? k_kv_append_q4<T, KV_MANY> : k_kv_append_q4<T, 1>, dim3((n + rows - 1) / rows), block, 0, c, (const T*)k, k_stride,
                      (const T*)v, v_stride, n, slots, positions, vec);
}

}  // namespace

cudaError_t launch_kv_append_q4(cudaStream_t st, const KvQ4& c, const void* k, size_t k_stride, const void* v, size_t v_stride, int dtype, int n,
                                const int32_t* slots, const int32_t* positions) {
    const size_t align = 4 * (size_t)dtype_bytes(dtype);
    const int vec = (((uintptr_t)k | (uintptr_t)v | k_stride * dtype_bytes(dtype) | v_stride * dtype_bytes(dtype)) & (align - 1)) == 0;
    auto* launch = dtype == DT_F32 ? launch_append<float> : dtype == DT_F16 ? launch_append<__half> : launch_append<__nv_bfloat16>;
    return launch(st, c, k, k_stride, v, v_stride, n, slots, positions, vec);
}

cudaError_t launch_kv_read_q4(cudaStream_t st, const KvQ4& c, int n, const int32_t* slots, const int32_t* positions, float* k, float* v) {
    const dim3 block = row_threads(c, 4);
    const unsigned rows = n >= KV_MANY_FROM ? KV_MANY * block.y : block.y;
    g_kernel_launches++;
    return launch_pdl(st, n >= KV_MANY_FROM ? k_kv_read_q4<KV_MANY> : k_kv_read_q4<1>, dim3((n + rows - 1) / rows), block, 0, c, n, slots, positions, k, v);
}

}  // namespace wick

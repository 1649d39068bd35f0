// Attention of single tokens over the 4-bit cache:  o = sum_t p_t V_t / sum_t p_t,  p_t = 2^(x_t - m),
// x_t = log2(e) / sqrt(d) q . K_t, with K_t and V_t blocks d (n - 8) of four-bit numbers n.
//
// Bound by HBM it would be 18 bytes per 32 elements of keys or values, 40 % of its time.  Most instructions are the unpacking (per 8 numbers one shift, four
// bit operations and four f16 ones); issue slots are 55 % busy (47 % with heads of 128): three warps to a scheduler (two), whose K part, softmax and V part
// follow one another, wait for their own results (of 4.2 cycles per instruction 1.1 for a fixed latency, 0.5 each for memory and for a busy pipe).
// f32 arithmetic on the CUDA cores would need 14
// operations per byte for 4 query heads, and an M = 128 tile of tcgen05 operands in shared memory that the CUDA cores would have to write.  So the
// products are mma.sync m16n8k16 with the numbers n - 8, exact in f16, as the 16-row operand.  The 8 columns of the other are 4 query
// heads: q, or the weights, is f32 and is held as two f16 parts (22 bits), the high one in an even column, the low one in the odd column behind it,
// so that the lane that gets both adds them.  (As rows of the 16-row operand, 4 heads left half of it empty: 1550 instead of 910 cycles per tile.)
//   scores:  S^T = sum over blocks of d_K ((n - 8) . q);  a block is two products, scaled and added in f32.
//   values:  O^T += (n - 8)^T (p d_V), per block; the weights' parts change from a lane per (key, head) to the operand's order by
//            movmatrix.  Sums over the 64 keys of a tile in the tensor core, over tiles in registers (with the running maximum's factor), since
//            the tensor core's additions truncate.
// High and low parts need a common exponent: q is scaled by a power of two per head, weights by one per tile, the largest |d_V| of
// the keys so far.
//
// Work: tiles of 64 keys of every (row, group of up to 8 query heads of a KV head), as one list that is cut into equal parts, first over the
// CTAs, then over their warps: any mix of lengths keeps every SM busy.  A warp streams its tiles through a ring of its own (four
// bulk copies per tile).  A (row, group) that lies within a warp's part is finished there, parts of one are joined within the CTA, and
// what reaches over CTAs goes to the workspace, where k_attention_q4_join adds it up in order: results do not depend on timing.
//
// On a B200: 64 rows of 1025 to 4100 keys, 32 / 8 heads of 64: 35 us (tensor pipe 15 %; the bytes would take 14); one row of 131,000 keys, 16 / 4 heads of 128:
// 28 us (8 warps fit the SM; bytes 12); one row of 517 keys, start, a tile and the join: 10 us.
//
// What lies behind a row's length is read (the tile is there) but not used: its scores are masked, its scales count as 0.
// Waits are bounded: on expiry the warp's outputs become NaN.
#include "serving.cuh"

namespace wick {

namespace {

constexpr int A4_TILE = KV_Q4_TILE, A4_HEADS = 8;
constexpr int A4_MIN_EXP = -24;  // of f16's smallest number

template <int NB>  // 32-element blocks of a head
struct Q4Cfg {
    static constexpr int HD = 32 * NB;
    static constexpr int QUANTS = A4_TILE * 16 * NB, SCALES = A4_TILE * 2 * NB;  // bytes of a tile
    static constexpr int STAGE = 2 * (QUANTS + SCALES);
    static constexpr int PART = A4_HEADS * HD + 2 * A4_HEADS;                    // floats of a partial result: o, m, l
    static constexpr int STAGES = 2;
    static constexpr int FIT = (218 * 1024) / (STAGES * STAGE + 2 * PART * 4), WARPS = FIT < 12 ? FIT : 12;
    // (Heads of 64: 10, 13, 14 warps took 40, 40, 37 us where 12 and 16 took 36: whole warps per scheduler.)
    static constexpr int THREADS = 32 * WARPS;
    static constexpr size_t SMEM = (size_t)WARPS * (STAGES * STAGE + 2 * PART * 4);
};

struct Q4Args {
    KvQ4 c;
    const void* q;
    size_t q_stride;
    const int32_t *slots, *lengths;
    void* out;
    int n, n_heads, group, sub, n_hg;  // query heads per KV head, head groups per KV head and in all
    int zero_rest;
    float scale_log2;
    ServingWaits waits;
    float* parts;   // [ctas][2][PART]: a CTA's part of what began before it, and of what goes on behind it
    int4* descs;    // [ctas][2]: row, head group, whether it holds its begin (1) and its end (2), whether there is one
};

__device__ __forceinline__ uint32_t s_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, uint32_t rounds) {
    for (uint32_t i = 0; i < rounds; i++)
        if (mbar_try_wait(bar, parity)) return true;
    return false;
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_zero(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {  // (a zero operand is no register)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {  // a in the low half
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
// Four-bit numbers at bits 0 and 16, or 4 and 20, of w as n - 8 in f16: 1024 + n is a number's bits behind f16's 1024.
__device__ __forceinline__ uint32_t behind_1024(uint32_t w, uint32_t mask) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "r"(mask), "r"(0x64006400u));  // (w & mask) | 1024s, in one
    return r;
}
__device__ __forceinline__ uint32_t low_pair(uint32_t w) {
    uint32_t r;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(behind_1024(w, 0x000F000Fu)), "r"(0xE408E408u));  // - 1032
    return r;
}
__device__ __forceinline__ uint32_t high_pair(uint32_t w) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(behind_1024(w, 0x00F000F0u)), "r"(0x2C002C00u), "r"(0xD480D480u));  // / 16 - 72
    return r;
}
// The high part of x, 11 bits.
__device__ __forceinline__ float high_part(float x) { return __uint_as_float(__float_as_uint(x) & 0xFFFFE000u); }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127

// The scales of a key's blocks in shared memory, as f32.
template <int NB>
__device__ __forceinline__ void load_scales(const __half* p, float (&d)[NB]) {
    if constexpr (NB == 2 || NB == 4) {
#pragma unroll
        for (int i = 0; i < NB; i += 2) {
            const float2 f = __half22float2(reinterpret_cast<const __half2*>(p)[i / 2]);
            d[i] = f.x, d[i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < NB; i++) d[i] = __half2float(p[i]);
    }
}

// The same, kept as they are: two to a register.
template <int NB>
__device__ __forceinline__ void load_packed(const __half* p, uint32_t (&w)[(NB + 1) / 2]) {
    if constexpr (NB % 2 == 0) {
#pragma unroll
        for (int i = 0; i < NB / 2; i++) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    } else {
        const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
        for (int i = 0; i < NB; i += 2) w[i / 2] = u[i] | (i + 1 < NB ? (uint32_t)u[i + 1 < NB ? i + 1 : 0] << 16 : 0u);
    }
}
__device__ __forceinline__ float half_of(uint32_t w, int i) { return __half2float(__ushort_as_half((unsigned short)(i & 1 ? w >> 16 : w & 0xFFFFu))); }

struct Cursor {  // a tile of the list
    int j, hg, t, tiles, len, slot;
};
__device__ __forceinline__ int row_tiles(const Q4Args& a, int j) {
    const int slot = a.slots[j], len = a.lengths[j];
    return slot < 0 || slot >= a.c.n_slots ? 0 : (max(0, min(len, a.c.max_seq)) + A4_TILE - 1) / A4_TILE;
}
__device__ __forceinline__ void enter_row(const Q4Args& a, Cursor& c) {
    c.slot = a.slots[c.j];
    c.len = max(0, min(a.lengths[c.j], a.c.max_seq));
    c.tiles = (c.len + A4_TILE - 1) / A4_TILE;
}
__device__ __forceinline__ void advance(const Q4Args& a, Cursor& c) {  // (the caller knows that there is another tile)
    if (++c.t < c.tiles) return;
    c.t = 0;
    if (++c.hg < a.n_hg) return;
    c.hg = 0;
    do c.j++;
    while (c.j < a.n - 1 && row_tiles(a, c.j) == 0);
    enter_row(a, c);
}

// The tiles ahead of the cursor, as running pointers: a tile costs four additions, another (row, head group) a look at the lists.
template <int NB>
struct Stream {
    using C = Q4Cfg<NB>;
    Cursor at;
    const uint8_t *kq, *vq;
    const __half *kd, *vd;
    __device__ __forceinline__ void place(const Q4Args& a) {
        const size_t row = a.c.row(at.slot, at.hg / a.sub, at.t * A4_TILE);
        kq = a.c.q[0] + row * (16 * NB), vq = a.c.q[1] + row * (16 * NB);
        kd = a.c.d[0] + row * NB, vd = a.c.d[1] + row * NB;
    }
    __device__ __forceinline__ void step(const Q4Args& a) {
        if (at.t + 1 < at.tiles) {
            at.t++;
            kq += C::QUANTS, vq += C::QUANTS, kd += C::SCALES / 2, vd += C::SCALES / 2;
        } else {
            advance(a, at);
            place(a);
        }
    }
    __device__ __forceinline__ void fetch(uint32_t stage, uint32_t bar) const {
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(C::STAGE) : "memory");
        bulk_copy(stage, kq, C::QUANTS, bar);
        bulk_copy(stage + C::QUANTS, vq, C::QUANTS, bar);
        bulk_copy(stage + 2 * C::QUANTS, kd, C::SCALES, bar);
        bulk_copy(stage + 2 * C::QUANTS + C::SCALES, vd, C::SCALES, bar);
    }
};

// An 8 x 8 matrix of 16-bit numbers, two of a row to a lane, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// One head of a chain of n parts, added up in order by a warp: its result, or, keep not null, the part that all of them are.  The maxima
// and sums are read by a lane per part, the weighted values eight parts at a time: a chain of dependent loads per part took 0.6 us each.
template <class T, int NB, class Part>
__device__ __forceinline__ void join_head(const Q4Args& a, int row, int hg, int g, int n, Part&& part, float* keep) {
    using C = Q4Cfg<NB>;
    const int lane = threadIdx.x & 31, head = hg / a.sub * a.group + hg % a.sub * A4_HEADS + g;
    float m = __int_as_float(0xFF800000);
    for (int k = lane; k < n; k += 32) m = fmaxf(m, part(k)[A4_HEADS * C::HD + g]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float l = 0.0f, o[NB] = {};
    for (int k0 = 0; k0 < n; k0 += 32) {
        float f = 0.0f;
        if (k0 + lane < n) {
            const float* p = part(k0 + lane);
            const float mi = p[A4_HEADS * C::HD + g];
            f = mi == m ? 1.0f : exp2_approx(mi - m);
            l = fmaf(p[A4_HEADS * C::HD + A4_HEADS + g], f, l);
        }
        for (int k = k0; k < min(n, k0 + 32); k += 8) {
            float x[8][NB];
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const float* p = part(min(k + u, n - 1)) + g * C::HD + lane;
#pragma unroll
                for (int b = 0; b < NB; b++) x[u][b] = p[32 * b];
            }
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const float w = __shfl_sync(0xffffffffu, f, (k - k0 + u) & 31);
                if (k + u < n) {
#pragma unroll
                    for (int b = 0; b < NB; b++) o[b] = fmaf(x[u][b], w, o[b]);
                }
            }
        }
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
    if (keep) {
#pragma unroll
        for (int b = 0; b < NB; b++) keep[g * C::HD + 32 * b + lane] = o[b];
        if (lane == 0) keep[A4_HEADS * C::HD + g] = m, keep[A4_HEADS * C::HD + A4_HEADS + g] = l;
    } else {
        const float inv = __fdiv_rn(1.0f, l);
        T* out = static_cast<T*>(a.out) + ((size_t)row * a.n_heads + head) * C::HD;
#pragma unroll
        for (int b = 0; b < NB; b++) out[32 * b + lane] = from_f32<T>(__fmul_rn(o[b], inv));
    }
}

// HQ: quads of query heads (1, or 2 for groups of 5 to 8).
template <class T, int NB, int HQ>
__global__ void __launch_bounds__(Q4Cfg<NB>::THREADS, 1) k_attention_q4(const __grid_constant__ Q4Args a) {
    using C = Q4Cfg<NB>;
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ __align__(8) unsigned long long bars[C::WARPS][C::STAGES];
    __shared__ unsigned long long pre[C::THREADS + 1];  // tiles of the rows before a thread's
    __shared__ unsigned long long warp_sum[C::WARPS];
    __shared__ int4 desc[C::WARPS][2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    if (lane < C::STAGES) asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(s_u32(&bars[warp][lane])), "r"(1 + a.waits.missing) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    if (lane < 2) desc[warp][lane] = make_int4(0, 0, 0, 0);
    pdl_trigger();
    pdl_wait();

    // ── where this CTA's and this warp's part of the list begins ──
    const int chunk = (a.n + C::THREADS - 1) / C::THREADS;
    unsigned long long mine = 0;
    for (int i = 0; i < chunk; i++) {
        const int j = tid * chunk + i;
        if (j < a.n) mine += row_tiles(a, j);
    }
    unsigned long long scan = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long v = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += v;
    }
    if (lane == 31) warp_sum[warp] = scan;
    __syncthreads();
    unsigned long long before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < C::WARPS; w++) {
        if (w < warp) before += warp_sum[w];
        total += warp_sum[w];
    }
    pre[tid] = before + scan - mine;
    __syncthreads();
    total *= (unsigned)a.n_hg;
    const unsigned long long ctas = total < gridDim.x ? total : gridDim.x;  // (a short list: one tile to a CTA)
    unsigned long long p0 = 0, p1 = 0;
    int working = 0;
    if (blockIdx.x < ctas) {
        const unsigned long long c0 = total * blockIdx.x / ctas, c1 = total * (blockIdx.x + 1) / ctas;
        const unsigned long long share = c1 - c0 < C::WARPS ? c1 - c0 : C::WARPS;  // (the first warps, where there are fewer tiles)
        working = (int)share;
        if (warp < working) p0 = c0 + (c1 - c0) * warp / share, p1 = c0 + (c1 - c0) * (warp + 1) / share;
    }
    float* parts = reinterpret_cast<float*>(sm + (size_t)C::WARPS * C::STAGES * C::STAGE);  // [warps][2][PART]
    bool ok = true;
    if (p0 < p1) {
        Cursor cur;
        {
            const unsigned long long row_at = p0 / (unsigned)a.n_hg;
            int lo = 0, hi = C::THREADS - 1;
            while (lo < hi) {  // the last thread whose rows begin at or before it
                const int mid = (lo + hi + 1) / 2;
                if (pre[mid] <= row_at) lo = mid;
                else hi = mid - 1;
            }
            unsigned long long acc = pre[lo];
            cur.j = lo * chunk;
            for (; cur.j < a.n - 1; cur.j++) {
                const int n = row_tiles(a, cur.j);
                if (acc + n > row_at) break;
                acc += n;
            }
            enter_row(a, cur);
            const unsigned long long r = p0 - acc * (unsigned)a.n_hg;
            cur.hg = (int)(r / (unsigned)cur.tiles), cur.t = (int)(r % (unsigned)cur.tiles);
        }
        const unsigned n_mine = (unsigned)(p1 - p0);
        uint8_t* ring = sm + (size_t)warp * C::STAGES * C::STAGE;
        const uint32_t ring_at = s_u32(ring), bars_at = s_u32(bars[warp]);
        Stream<NB> ahead;
        ahead.at = cur;
        ahead.place(a);
        unsigned fetched = 0;
        for (; fetched < C::STAGES && fetched < n_mine; fetched++) {
            if (fetched) ahead.step(a);
            if (lane == 0) ahead.fetch(ring_at + fetched * C::STAGE, bars_at + fetched * 8);
        }
        uint32_t qb[HQ][NB][2][2];  // column g: head g / 2 of the quad, its high (g even) or low part
        float q_inv[HQ], m[HQ], l[HQ], o[HQ][NB][2][2];  // of head t4 of the quad; o: dims 16 h + 2 g + e of a block as [h][e]
        int vexp = A4_MIN_EXP;   // l and o are scaled by 2^(12 - vexp)
        bool begins = false, fresh = true;
        for (unsigned i = 0; i < n_mine; i++) {
            if (fresh) {  // another row or head group
                fresh = false;
                begins = cur.t == 0;
                vexp = A4_MIN_EXP;
                const int h0 = cur.hg % a.sub * A4_HEADS;
#pragma unroll
                for (int u = 0; u < HQ; u++) {
                    m[u] = __int_as_float(0xFF800000), l[u] = 0.0f;
#pragma unroll
                    for (int b = 0; b < NB; b++) o[u][b][0][0] = o[u][b][0][1] = o[u][b][1][0] = o[u][b][1][1] = 0.0f;
                    const int h = h0 + 4 * u + (g >> 1);
                    const bool real = h < a.group;
                    const T* q = static_cast<const T*>(a.q) + (size_t)cur.j * a.q_stride + (size_t)((cur.hg / a.sub) * a.group + (real ? h : 0)) * C::HD;
                    float x[NB][2][4], top = 0.0f;
#pragma unroll
                    for (int b = 0; b < NB; b++)
#pragma unroll
                        for (int k = 0; k < 2; k++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                x[b][k][e] = real ? __fmul_rn(to_f32(q[32 * b + 16 * k + 4 * t4 + e]), a.scale_log2) : 0.0f;
                                top = fmaxf(top, fabsf(x[b][k][e]));
                            }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const int e = max(-100, min(127, (int)((__float_as_uint(top) >> 23) & 255u) - 127));
                    const float f = pow2(12 - e);
                    q_inv[u] = __shfl_sync(0xffffffffu, pow2(e - 12), 8 * t4);  // (from the lanes of column 2 t4)
#pragma unroll
                    for (int b = 0; b < NB; b++)
#pragma unroll
                        for (int s = 0; s < 2; s++)
#pragma unroll
                            for (int k = 0; k < 2; k++) {
                                const float x0 = __fmul_rn(x[b][k][s], f), x1 = __fmul_rn(x[b][k][2 + s], f), y0 = high_part(x0), y1 = high_part(x1);
                                qb[u][b][s][k] = (g & 1) ? pack_f16(__fsub_rn(x0, y0), __fsub_rn(x1, y1)) : pack_f16(y0, y1);
                            }
                }
            }
            const unsigned st = i % C::STAGES;
            if (ok) ok = __all_sync(0xffffffffu, bar_wait(bars_at + st * 8, (i / C::STAGES) & 1, a.waits.rounds));  // (the warp's answer: all its outputs or none)
            const uint8_t* stage = ring + st * C::STAGE;
            const uint32_t* kw = reinterpret_cast<const uint32_t*>(stage);
            const uint32_t* vw = reinterpret_cast<const uint32_t*>(stage + C::QUANTS);
            const __half* kd = reinterpret_cast<const __half*>(stage + 2 * C::QUANTS);
            const __half* vd = reinterpret_cast<const __half*>(stage + 2 * C::QUANTS + C::SCALES);
            const int seen = cur.len - cur.t * A4_TILE;
            // Row g of the 8-key half e of a block of 16 keys is its key g / 2 + 4 (g & 1) + 8 e: a lane then reads the values of rows 2 t4 and
            // 2 t4 + 1 without bank conflicts.
            const int key_g = (g >> 1) + 4 * (g & 1);
            float s[HQ][4][2];
            constexpr int NW = (NB + 1) / 2;
            uint32_t dv[4][2][NW];
#pragma unroll
            for (int b16 = 0; b16 < 4; b16++) {
                float d0[NB], d1[NB], sum[HQ][2];
                const int key = 16 * b16 + key_g;
                load_scales<NB>(kd + key * NB, d0);
                load_scales<NB>(kd + (key + 8) * NB, d1);
                load_packed<NB>(vd + key * NB, dv[b16][0]);
                load_packed<NB>(vd + (key + 8) * NB, dv[b16][1]);
#pragma unroll
                for (int u = 0; u < HQ; u++) sum[u][0] = sum[u][1] = 0.0f;
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const uint32_t w0 = kw[key * 4 * NB + 4 * b + t4], w1 = kw[(key + 8) * 4 * NB + 4 * b + t4];
                    const uint32_t k0[4] = {low_pair(w0), low_pair(w1), high_pair(w0), high_pair(w1)};
                    const uint32_t k1[4] = {low_pair(w0 >> 8), low_pair(w1 >> 8), high_pair(w0 >> 8), high_pair(w1 >> 8)};
#pragma unroll
                    for (int u = 0; u < HQ; u++) {
                        float c[4];
                        mma16816_zero(c, k0, qb[u][b][0][0], qb[u][b][0][1]);
                        mma16816(c, k1, qb[u][b][1][0], qb[u][b][1][1]);
                        sum[u][0] = fmaf(__fadd_rn(c[0], c[1]), d0[b], sum[u][0]);
                        sum[u][1] = fmaf(__fadd_rn(c[2], c[3]), d1[b], sum[u][1]);
                    }
                }
#pragma unroll
                for (int u = 0; u < HQ; u++) s[u][b16][0] = sum[u][0], s[u][b16][1] = sum[u][1];
            }
            if (seen < A4_TILE) {  // the row's last tile
#pragma unroll
                for (int b16 = 0; b16 < 4; b16++)
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        if (16 * b16 + 8 * e + key_g >= seen) {
#pragma unroll
                            for (int u = 0; u < HQ; u++) s[u][b16][e] = __int_as_float(0xFF800000);
#pragma unroll
                            for (int b = 0; b < NW; b++) dv[b16][e][b] = 0;
                        }
            }
            __half2 vmax = __float2half2_rn(0.0f);
#pragma unroll
            for (int b16 = 0; b16 < 4; b16++)
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int b = 0; b < NW; b++) vmax = __hmax2(vmax, __habs2(*reinterpret_cast<__half2*>(&dv[b16][e][b])));
            float vtop = fmaxf(__low2float(vmax), __high2float(vmax));
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, x));
            const int old = vexp;
            vexp = max(vexp, min((int)((__float_as_uint(vtop) >> 23) & 255u) - 127, 16));  // (not finite: 16)
            const float moved = pow2(old - vexp);
            float keep[HQ];
#pragma unroll
            for (int u = 0; u < HQ; u++) {
                float top = fmaxf(s[u][0][0], s[u][0][1]);
#pragma unroll
                for (int b16 = 1; b16 < 4; b16++) top = fmaxf(top, fmaxf(s[u][b16][0], s[u][b16][1]));
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                top = fmaxf(m[u], __fmul_rn(top, q_inv[u]));
                keep[u] = __fmul_rn(m[u] == top ? 1.0f : exp2_approx(m[u] - top), moved);
                m[u] = top;
                // (two additions: a large maximum would swallow the power of two; the product with q_inv is exact)
                const float from = top == __int_as_float(0xFF800000) ? 0.0f : -top, lift = (float)(12 - vexp);
                float sum = 0.0f;
#pragma unroll
                for (int b16 = 0; b16 < 4; b16++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        s[u][b16][e] = exp2_approx(__fadd_rn(fmaf(s[u][b16][e], q_inv[u], from), lift));
                        sum = __fadd_rn(sum, s[u][b16][e]);
                    }
                l[u] = fmaf(l[u], keep[u], sum);
            }
            const uint32_t half_sel = (g & 1) ? 0x7632u : 0x5410u;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                float acc[HQ][2][4];
#pragma unroll
                for (int b16 = 0; b16 < 4; b16++) {
                    uint32_t r[2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int key = 16 * b16 + 8 * e + t4;
                        r[e] = __byte_perm(vw[key * 4 * NB + 4 * b + (g >> 1)], vw[(key + 4) * 4 * NB + 4 * b + (g >> 1)], half_sel);
                    }
                    const uint32_t v0[4] = {low_pair(r[0]), high_pair(r[0]), low_pair(r[1]), high_pair(r[1])};                          // dims 2 g, 16 + 2 g
                    const uint32_t v1[4] = {low_pair(r[0] >> 8), high_pair(r[0] >> 8), low_pair(r[1] >> 8), high_pair(r[1] >> 8)};  // and the next ones
#pragma unroll
                    for (int u = 0; u < HQ; u++) {
                        uint32_t pb[2];
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const float x = __fmul_rn(s[u][b16][e], half_of(dv[b16][e][b / 2], b)), y = high_part(x);
                            pb[e] = transposed(pack_f16(y, __fsub_rn(x, y)));
                        }
                        if (b16 == 0) {
                            mma16816_zero(acc[u][0], v0, pb[0], pb[1]);
                            mma16816_zero(acc[u][1], v1, pb[0], pb[1]);
                        } else {
                            mma16816(acc[u][0], v0, pb[0], pb[1]);
                            mma16816(acc[u][1], v1, pb[0], pb[1]);
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < HQ; u++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        o[u][b][0][e] = fmaf(o[u][b][0][e], keep[u], __fadd_rn(acc[u][e][0], acc[u][e][1]));
                        o[u][b][1][e] = fmaf(o[u][b][1][e], keep[u], __fadd_rn(acc[u][e][2], acc[u][e][3]));
                    }
            }
            __syncwarp();  // every lane has read the stage
            if (fetched < n_mine) {
                ahead.step(a);
                if (lane == 0 && ok) ahead.fetch(ring_at + st * C::STAGE, bars_at + st * 8);
                fetched++;
            }
            const bool ends = cur.t + 1 == cur.tiles;
            if (ends || i + 1 == n_mine) {
                const float down = pow2(vexp - 12);
                const int h0 = cur.hg % a.sub * A4_HEADS;
                const bool whole = begins && ends;
                const int place = begins ? 1 : 0;
                float* part = parts + (warp * 2 + place) * C::PART;
#pragma unroll
                for (int u = 0; u < HQ; u++) {
                    const int h = 4 * u + t4;
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) l[u] += __shfl_xor_sync(0xffffffffu, l[u], x);
                    if (!ok) l[u] = __int_as_float(0x7FC00000);
                    if (whole) {
                        if (h0 + h < a.group) {
                            const float inv = __fdiv_rn(1.0f, l[u]);
                            T* out = static_cast<T*>(a.out) + ((size_t)cur.j * a.n_heads + (cur.hg / a.sub) * a.group + h0 + h) * C::HD + 2 * g;
#pragma unroll
                            for (int b = 0; b < NB; b++)
#pragma unroll
                                for (int k = 0; k < 2; k++) {
                                    out[32 * b + 16 * k] = from_f32<T>(__fmul_rn(o[u][b][k][0], inv));
                                    out[32 * b + 16 * k + 1] = from_f32<T>(__fmul_rn(o[u][b][k][1], inv));
                                }
                        }
                    } else {
#pragma unroll
                        for (int b = 0; b < NB; b++)
#pragma unroll
                            for (int k = 0; k < 2; k++) {
                                part[h * C::HD + 32 * b + 16 * k + 2 * g] = __fmul_rn(o[u][b][k][0], down);
                                part[h * C::HD + 32 * b + 16 * k + 2 * g + 1] = __fmul_rn(o[u][b][k][1], down);
                            }
                        if (g == 0) part[A4_HEADS * C::HD + h] = m[u], part[A4_HEADS * C::HD + A4_HEADS + h] = __fmul_rn(l[u], down);
                    }
                }
                if (!whole && lane == 0) desc[warp][place] = make_int4(cur.j, cur.hg, (begins ? 1 : 0) | (ends ? 2 : 0), 1);
                fresh = true;
            }
            if (i + 1 < n_mine) advance(a, cur);
        }
    }
    // rows without a tile: zeros where the row is one of the cache (or zero_rest asks for it)
    for (int j = blockIdx.x; j < a.n; j += gridDim.x)
        if (row_tiles(a, j) == 0 && (a.zero_rest || (a.slots[j] >= 0 && a.slots[j] < a.c.n_slots)))
            for (int i = tid; i < a.n_heads * C::HD; i += C::THREADS) static_cast<T*>(a.out)[(size_t)j * a.n_heads * C::HD + i] = from_f32<T>(0.0f);
    if (tid < 2) a.descs[(size_t)blockIdx.x * 2 + tid] = make_int4(0, 0, 0, 0);
    if (!ok) settle();  // (copies may still be landing)
    __syncthreads();

    // ── parts within the CTA.  A chain starts with the part that begins in a warp (place 1) or with the first part of all, if that began
    //    before the CTA, and goes on with the parts that began before (place 0) of the warps behind, up to the one that holds the end. ──
    const bool has0 = lane < C::WARPS && desc[lane < C::WARPS ? lane : 0][0].w, has1 = lane < C::WARPS && desc[lane < C::WARPS ? lane : 0][1].w;
    const uint32_t valid0 = __ballot_sync(0xffffffffu, has0), valid1 = __ballot_sync(0xffffffffu, has1);
    const uint32_t end0 = __ballot_sync(0xffffffffu, has0 && (desc[lane < C::WARPS ? lane : 0][0].z & 2));
    const int opening = valid0 ? __ffs(valid0) - 1 : C::WARPS;  // the warp whose part began before the CTA
    const bool opens = valid0 && !(valid1 & ((1u << opening) - 1));
    const int chains = __popc(valid1) + (opens ? 1 : 0);
    for (int item = warp; item < chains * A4_HEADS; item += C::WARPS) {
        const int g8 = item % A4_HEADS, c = item / A4_HEADS - (opens ? 1 : 0), place = c < 0 ? 0 : 1;
        const int first = c < 0 ? opening : __fns(valid1, 0, c + 1);
        const int4 d = desc[first][place];
        if (d.y % a.sub * A4_HEADS + g8 >= a.group) continue;
        const uint32_t ends = place == 0 ? end0 >> first << first : first == 31 ? 0 : end0 >> (first + 1) << (first + 1);
        const int last = ends ? __ffs(ends) - 1 : working - 1;
        const int flags = (place ? 1 : 0) | (ends ? 2 : 0);
        const size_t to = (size_t)blockIdx.x * 2 + place;
        join_head<T, NB>(a, d.x, d.y, g8, last - first + 1, [&](int k) { return parts + ((first + k) * 2 + (k == 0 ? place : 0)) * C::PART; },
                         flags == 3 ? nullptr : a.parts + to * C::PART);
        if (flags != 3 && g8 == 0 && lane == 0) a.descs[to] = make_int4(d.x, d.y, flags, 1);
    }
}

// What reaches over CTAs: CTA (b, g) joins head g of what begins in CTA b of the kernel above and goes on.  Its warps take the parts in turn, and
// warp 0 adds up their sums in the warps' order.
constexpr int JOIN_WARPS = 8;
template <class T, int NB>
__global__ void __launch_bounds__(32 * JOIN_WARPS) k_attention_q4_join(const __grid_constant__ Q4Args a) {
    using C = Q4Cfg<NB>;
    __shared__ float sums[JOIN_WARPS][C::HD + 2];
    pdl_trigger();
    pdl_wait();
    const int4 d = a.descs[(size_t)blockIdx.x * 2 + 1];
    const int g = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (!d.w || d.y % a.sub * A4_HEADS + g >= a.group) return;
    int last = blockIdx.x;  // the CTA that holds the end
    for (int b = blockIdx.x + 1;; b += 32) {
        const bool in = b + lane < (int)gridDim.x;
        const uint32_t end = __ballot_sync(0xffffffffu, in && (a.descs[(size_t)(b + lane) * 2].z & 2));
        if (end) {
            last = b + __ffs(end) - 1;
            break;
        }
        if (b + 32 >= (int)gridDim.x) return;  // (cannot be)
    }
    const float* first = a.parts + ((size_t)blockIdx.x * 2 + 1) * C::PART;
    const int n = last - (int)blockIdx.x + 1, mine = (n - warp + JOIN_WARPS - 1) / JOIN_WARPS;
    auto part = [&](int k) { return first + (k == 0 ? 0 : (k * 2 - 1) * C::PART); };
    if (n <= 4) {
        if (warp == 0) join_head<T, NB>(a, d.x, d.y, g, n, part, nullptr);
        return;
    }
    float m = __int_as_float(0xFF800000), l = 0.0f, o[NB] = {};
    for (int k0 = 0; k0 < mine; k0 += 8) {  // eight parts' loads together; rescaled where a maximum grows
        float x[8][NB], mi[8], li[8];
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const float* p = part(min(warp + (k0 + u) * JOIN_WARPS, n - 1));
            const bool in = k0 + u < mine;
            mi[u] = in ? p[A4_HEADS * C::HD + g] : __int_as_float(0xFF800000);
            li[u] = p[A4_HEADS * C::HD + A4_HEADS + g];
#pragma unroll
            for (int b = 0; b < NB; b++) x[u][b] = p[g * C::HD + 32 * b + lane];
        }
        float top = m;
#pragma unroll
        for (int u = 0; u < 8; u++) top = fmaxf(top, mi[u]);
        const float f0 = m == top ? 1.0f : exp2_approx(m - top);
        l *= f0;
#pragma unroll
        for (int b = 0; b < NB; b++) o[b] *= f0;
#pragma unroll
        for (int u = 0; u < 8; u++)
            if (k0 + u < mine) {
                const float f = mi[u] == top ? 1.0f : exp2_approx(mi[u] - top);
                l = fmaf(li[u], f, l);
#pragma unroll
                for (int b = 0; b < NB; b++) o[b] = fmaf(x[u][b], f, o[b]);
            }
        m = top;
    }
#pragma unroll
    for (int b = 0; b < NB; b++) sums[warp][32 * b + lane] = o[b];
    if (lane == 0) sums[warp][C::HD] = m, sums[warp][C::HD + 1] = l;
    __syncthreads();
    if (warp != 0) return;
    m = __int_as_float(0xFF800000);
    for (int w = 0; w < JOIN_WARPS; w++) m = fmaxf(m, sums[w][C::HD]);
    l = 0.0f;
#pragma unroll
    for (int b = 0; b < NB; b++) o[b] = 0.0f;
    for (int w = 0; w < JOIN_WARPS && w < n; w++) {
        const float f = sums[w][C::HD] == m ? 1.0f : exp2_approx(sums[w][C::HD] - m);
        l = fmaf(sums[w][C::HD + 1], f, l);
#pragma unroll
        for (int b = 0; b < NB; b++) o[b] = fmaf(sums[w][32 * b + lane], f, o[b]);
    }
    const float inv = __fdiv_rn(1.0f, l);
    T* out = static_cast<T*>(a.out) + ((size_t)d.x * a.n_heads + d.y / a.sub * a.group + d.y % a.sub * A4_HEADS + g) * C::HD;
#pragma unroll
    for (int b = 0; b < NB; b++) out[32 * b + lane] = from_f32<T>(__fmul_rn(o[b], inv));
}

constexpr int A4_MAX_CTAS = 256;
size_t part_bytes(int head_dim) { return (size_t)A4_MAX_CTAS * 2 * (A4_HEADS * head_dim + 2 * A4_HEADS) * sizeof(float); }

template <class T, int NB, int HQ>
cudaError_t launch_quads(cudaStream_t st, Q4Args& a) {
    using C = Q4Cfg<NB>;
    static RaisedPerDevice limit;
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if ((e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return e;
    if ((e = raise_dynamic_smem(limit, (const void*)k_attention_q4<T, NB, HQ>, C::SMEM)) != cudaSuccess) return e;
    const dim3 grid((unsigned)(sms < A4_MAX_CTAS ? sms : A4_MAX_CTAS));
    g_kernel_launches += 2;
    if ((e = launch_pdl(st, k_attention_q4<T, NB, HQ>, grid, dim3(C::THREADS), C::SMEM, a)) != cudaSuccess) return e;
    return launch_pdl(st, k_attention_q4_join<T, NB>, dim3(grid.x, (unsigned)(a.group < A4_HEADS ? a.group : A4_HEADS)), dim3(32 * JOIN_WARPS), 0, a);
}
template <class T, int NB>
cudaError_t launch_typed(cudaStream_t st, Q4Args& a) {
    return a.group <= 4 ? launch_quads<T, NB, 1>(st, a) : launch_quads<T, NB, 2>(st, a);
}
template <class T>
cudaError_t launch_head(cudaStream_t st, Q4Args& a) {
    switch (a.c.head_dim / QK) {
        case 1: return launch_typed<T, 1>(st, a);
        case 2: return launch_typed<T, 2>(st, a);
        case 3: return launch_typed<T, 3>(st, a);
        default: return launch_typed<T, 4>(st, a);
    }
}

}  // namespace

size_t attention_q4_workspace(int head_dim) { return part_bytes(head_dim) + A4_MAX_CTAS * 2 * sizeof(int4); }

cudaError_t launch_attention_q4(cudaStream_t st, const KvQ4& c, const void* q, size_t q_stride, int dtype, int n, int n_heads, const int32_t* slots,
                                const int32_t* lengths, void* out, int zero_rest, void* workspace) {
    Q4Args a{};
    a.c = c;
    a.q = q, a.q_stride = q_stride;
    a.slots = slots, a.lengths = lengths;
    a.out = out;
    a.n = n, a.n_heads = n_heads, a.group = n_heads / c.n_kv, a.sub = (a.group + A4_HEADS - 1) / A4_HEADS, a.n_hg = c.n_kv * a.sub;
    a.zero_rest = zero_rest;
    a.waits = serving_waits();
    a.scale_log2 = 1.4426950408889634f / sqrtf((float)c.head_dim);
    a.parts = static_cast<float*>(workspace);
    a.descs = reinterpret_cast<int4*>(static_cast<uint8_t*>(workspace) + part_bytes(c.head_dim));
    return dtype == DT_F32 ? launch_head<float>(st, a) : dtype == DT_F16 ? launch_head<__half>(st, a) : launch_head<__nv_bfloat16>(st, a);
}

}  // namespace wick

// Causal attention of packed prompts with grouped heads on tcgen05.
//
// Token j of a sequence with nq tokens and nk keys attends its keys t <= j + nk - nq:  o_j = sum_t p_t v_t / sum_t p_t with
// p_t = 2^(x_t - m), x_t = log2(e) / sqrt(d) q_j . k_t, m a running maximum.
//
// A CTA takes 2 x 128 rows of one KV head: a row is a (token, query head of the group) pair, 128 / group tokens to a tile, so that a K / V tile
// that lies in shared memory serves every head of its group and short prompts fill the rows.  K and V tiles of NK keys go through one ring
// of TMA slots (K0 V0 K1 V1 ..).  Per row tile: S = Q K^T (tcgen05, S in tensor memory) -> the tile's four softmax warps, one row per
// thread -> P over S in tensor memory -> P V with P as the A operand from there.  The two row tiles alternate: while one is in the
// tensor core the other is in its softmax.
//
// f16, bf16: one product each; O stays in tensor memory, and is rescaled only where a row's maximum has grown by more than 2^8 (a weight is at
//   most 2^8 then; the last maximum that was used cancels in the quotient).
// f32: every operand is split into two f16 parts, x = 2^e (hi + lo), 22 bits, with one power of two per row of Q and per tile of K and V
//   (k_split), and a product is hi hi + hi lo + lo hi (lo lo is 2^-22 of it).  The tensor core adds with truncation, so that a sum over
//   thousands of keys would drift by 1e-5: O is taken out after every tile and added up in registers.
//
// Masked places may hold anything.  Scores are masked after the product; V is different, 0 * NaN is NaN: a warp looks at every V
// tile that some row sees in part, zeroes what is not finite, and notes the keys; rows that attend such a key add its values at the end.
//
// Every wait is bounded: on expiry all roles leave their loops and the rows of the CTA become NaN.
#include <cuda.h>
#include <algorithm>
#include <mutex>

#include "serving.cuh"

namespace wick {

namespace {

constexpr int PR_ROWS = 128;      // rows of a tile == lanes of tensor memory
constexpr int PR_THREADS = 384;   // TMA, MMA, V check, idle; 2 x 4 softmax warps
constexpr int PR_MASKED = 8;      // tiles that some row of a CTA sees in part: at most 256 / 64 + 2
constexpr int PR_ZERO_CTAS = 32;
constexpr uint32_t PR_SPIN_LIMIT = 1u << 18;  // try_wait suspends for a while: of the order of a second
constexpr float PR_LAZY = 8.0f;

template <int PLANES, int HDP>
struct Cfg {
    static constexpr int NK = PLANES == 2 && HDP == 128 ? 64 : 128;  // keys of a tile
    static constexpr int CH = HDP / 64;                              // 128-byte columns of a row
    static constexpr int QBYTES = PR_ROWS * 128 * CH;                // a plane of a Q tile
    static constexpr int KBYTES = NK * 128 * CH;                     // a plane of a K or V tile
    static constexpr int SLOT = PLANES * KBYTES;
    static constexpr int FIT = (225 * 1024 - 2 * PLANES * QBYTES) / SLOT, NS = FIT < 6 ? FIT : 6;
    static constexpr bool O_IN_TMEM = PLANES == 1;
    static constexpr int O_BUFS = PLANES == 2 && HDP == 64 ? 2 : 1;
    static constexpr int S_COL = 0, O_COL = NK;                      // columns of a row tile's 256
    static_assert(NK + O_BUFS * HDP <= 256 && NS >= 3, "tensor or shared memory");
    static constexpr size_t SMEM = 1024 + (size_t)2 * PLANES * QBYTES + (size_t)NS * SLOT + 1024;
};

struct Barriers {
    unsigned long long q_full, full[6], empty[6], ready[6], s_full[2], p_ready[2], checked[PR_MASKED];
    uint32_t mask[PR_MASKED][4];
    uint32_t tmem_base;
    volatile uint32_t abort;
};

// What the kernels read besides the tensor maps.
struct PromptArgs {
    Prompts p;
    const float *q_inv, *k_inv, *v_inv;  // f32: the powers of two taken out of q rows and K / V tiles
    int group, tile_tokens;              // query heads per KV head, tokens of a row tile
    int slots;                           // places for (sequence, block of 2 * tile_tokens tokens)
    int zero_rest;
    float scale_log2;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(void* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(void* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void bar_expect(void* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(void* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
// false: the limit, or another role has given up
__device__ __forceinline__ bool bar_wait(Barriers* b, void* bar, uint32_t parity) {
    for (uint32_t i = 0; i < PR_SPIN_LIMIT; i++) {
        if (bar_try(bar, parity)) return true;
        if ((i & 255u) == 255u && b->abort) return false;
    }
    b->abort = 1;
    return false;
}
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p;
}
__device__ __forceinline__ void tma_4d(uint32_t dst, const CUtensorMap* map, void* bar, int x, int head, int row, int plane) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"((unsigned long long)map), "r"(smem_u32(bar)), "r"(x), "r"(head), "r"(row), "r"(plane)
        : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void umma_commit(void* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Operand rows of 128 bytes in 128-byte swizzle.  K-major (Q, K): 8-row atoms 1024 bytes apart.  MN-major (V): atoms of 64 columns x 8
// keys, 1024 bytes from 8 keys to the next, `lead` bytes from 64 columns to the next.
__device__ __forceinline__ unsigned long long umma_desc(uint32_t addr, uint32_t lead) {
    return (unsigned long long)((addr >> 4) & 0x3FFF) | (unsigned long long)((lead >> 4) & 0x3FFF) << 16 | (unsigned long long)(1024 >> 4) << 32 |
           1ull << 46 | 2ull << 61;
}
__device__ __forceinline__ void umma_ss(uint32_t d, unsigned long long a, unsigned long long b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add)
        : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, unsigned long long b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(add)
        : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]),
          "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]),
          "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]),
          "=f"(r[31])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const float* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"f"(r[0]),
        "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]), "f"(r[8]), "f"(r[9]), "f"(r[10]), "f"(r[11]), "f"(r[12]),
        "f"(r[13]), "f"(r[14]), "f"(r[15]), "f"(r[16]), "f"(r[17]), "f"(r[18]), "f"(r[19]), "f"(r[20]), "f"(r[21]), "f"(r[22]), "f"(r[23]),
        "f"(r[24]), "f"(r[25]), "f"(r[26]), "f"(r[27]), "f"(r[28]), "f"(r[29]), "f"(r[30]), "f"(r[31]), "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
        "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <class T>
__device__ __forceinline__ uint32_t pack16(float a, float b) {  // a in the low half
    uint32_t r;
    if constexpr (sizeof(T) == 2 && !std::is_same<T, __nv_bfloat16>::value)
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    else
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

// The sequence whose places hold `slot`: sequence s has the places floor(starts[s] / block) + s .. of its blocks, which never overlap.
// Called by a whole warp; -1: none.
__device__ __forceinline__ int find_seq(const int32_t* starts, int n_seqs, int n_rows, int block, int slot) {
    const int lane = threadIdx.x & 31;
    auto place = [&](int s) { return max(0, min(starts[s], n_rows)) / block + s; };
    int lo = 0, n = n_seqs;
    while (true) {
        const int step = (n + 31) / 32, s = lo + lane * step;
        const bool at = lane * step < n && s < n_seqs && place(s) <= slot;
        const int count = __popc(__ballot_sync(0xffffffffu, at));
        if (count == 0) return -1;
        lo += (count - 1) * step;
        if (step == 1) return lo;
        n = step;
    }
}

struct Block {  // the rows of a CTA
    int token0, tokens;  // first token (a row of q), tokens of the block
    int key0, keys;      // first key (a row of k), keys of the sequence
    int first_visible;   // keys that the block's first token attends (may be negative)
    __device__ __forceinline__ int visible(int j) const { return max(0, min(first_visible + j, keys)); }
};

template <class T, int PLANES, int HDP>
__global__ void __launch_bounds__(PR_THREADS, 1)
k_attention_prompts(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                    const __grid_constant__ PromptArgs a) {
    using C = Cfg<PLANES, HDP>;
    using T16 = typename std::conditional<PLANES == 2, __half, T>::type;
    constexpr int NK = C::NK, NS = C::NS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    Barriers* bar = reinterpret_cast<Barriers*>(sm + 2 * PLANES * C::QBYTES + NS * C::SLOT);
    const uint32_t q_smem = smem_u32(sm), ring = q_smem + 2 * PLANES * C::QBYTES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hd = a.p.head_dim;
    pdl_trigger();
    pdl_wait();

    if ((int)blockIdx.x >= a.slots * a.p.n_kv) {  // rows of no sequence
        const int first = max(0, min(a.p.starts[0], a.p.n_tokens)), last = max(first, min(a.p.starts[a.p.n_seqs], a.p.n_tokens));
        const size_t row = (size_t)a.p.n_heads * hd * sizeof(T) / 16, n = (size_t)(a.p.n_tokens - last + first) * row;
        for (size_t i = (size_t)(blockIdx.x - a.slots * a.p.n_kv) * PR_THREADS + threadIdx.x; i < n; i += (size_t)PR_ZERO_CTAS * PR_THREADS)
            reinterpret_cast<uint4*>(a.p.out)[i < first * row ? i : i + (size_t)(last - first) * row] = make_uint4(0, 0, 0, 0);
        return;
    }
    // The last places first: a sequence's last blocks have the most keys, and the launch then ends with short ones.
    const int slot = a.slots - 1 - (int)blockIdx.x / a.p.n_kv, kvh = (int)blockIdx.x % a.p.n_kv;
    const int seq = find_seq(a.p.starts, a.p.n_seqs, a.p.n_tokens, 2 * a.tile_tokens, slot);
    if (seq < 0) return;
    Block blk;
    int key_slot0;
    {
        const int32_t* ks = a.p.key_starts ? a.p.key_starts : a.p.starts;
        const int q0 = max(0, min(a.p.starts[seq], a.p.n_tokens)), q1 = max(q0, min(a.p.starts[seq + 1], a.p.n_tokens));
        const int k0 = max(0, min(ks[seq], a.p.n_keys)), k1 = max(k0, min(ks[seq + 1], a.p.n_keys));
        const int at = (slot - (q0 / (2 * a.tile_tokens) + seq)) * 2 * a.tile_tokens;
        if (at >= q1 - q0) return;
        blk.token0 = q0 + at;
        blk.tokens = min(2 * a.tile_tokens, q1 - blk.token0);
        blk.key0 = k0, blk.keys = k1 - k0;
        blk.first_visible = at + 1 + blk.keys - (q1 - q0);
        key_slot0 = k0 / NK + seq;
    }
    // tiles of keys that the two row tiles see
    int n_tiles[2];
#pragma unroll
    for (int m = 0; m < 2; m++) {
        const int rows = min(a.tile_tokens, blk.tokens - m * a.tile_tokens);
        n_tiles[m] = rows > 0 ? (blk.visible(m * a.tile_tokens + rows - 1) + NK - 1) / NK : 0;
    }
    const int nt = max(n_tiles[0], n_tiles[1]);
    const int first_masked = max(0, blk.first_visible) / NK;  // tiles from here on are seen in part by some row

    if (threadIdx.x == 0) {
        bar_init(&bar->q_full, 1);
        for (int s = 0; s < NS; s++) bar_init(&bar->full[s], 1), bar_init(&bar->empty[s], 1), bar_init(&bar->ready[s], 1);
        for (int m = 0; m < 2; m++) bar_init(&bar->s_full[m], 1), bar_init(&bar->p_ready[m], 4);
        for (int i = 0; i < PR_MASKED; i++) bar_init(&bar->checked[i], 1);
        bar->abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bar->tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bar->tmem_base;

    if (warp == 0) {
        // ── TMA ──────────────────────────────────────────────────────────────
        if (lane == 0 && nt > 0) {
            const int tiles_q = n_tiles[1] > 0 ? 2 : 1;
            bar_expect(&bar->q_full, (uint32_t)(tiles_q * PLANES * C::CH * a.group * a.tile_tokens * 128));
            for (int m = 0; m < tiles_q; m++)
                for (int p = 0; p < PLANES; p++)
                    for (int c = 0; c < C::CH; c++)
                        tma_4d(q_smem + (m * PLANES + p) * C::QBYTES + c * PR_ROWS * 128, &map_q, &bar->q_full, c * 64, kvh * a.group,
                               blk.token0 + m * a.tile_tokens, p);
            for (int g = 0; g < 2 * nt; g++) {
                const int s = g % NS, u = g / NS;
                if (!bar_wait(bar, &bar->empty[s], (u & 1) ^ 1)) break;
                bar_expect(&bar->full[s], C::SLOT);
                for (int p = 0; p < PLANES; p++)
                    for (int c = 0; c < C::CH; c++)
                        tma_4d(ring + s * C::SLOT + p * C::KBYTES + c * NK * 128, (g & 1) ? &map_v : &map_k, &bar->full[s], c * 64, kvh,
                               blk.key0 + (g >> 1) * NK, p);
            }
        }
    } else if (warp == 1) {
        // ── MMA ──────────────────────────────────────────────────────────────
        const uint32_t leader = elect_one();
        constexpr uint32_t type = std::is_same<T16, __nv_bfloat16>::value ? 1u : 0u;
        constexpr uint32_t idesc_s = (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)(NK >> 3) << 17) | ((uint32_t)(PR_ROWS >> 4) << 24);
        constexpr uint32_t idesc_o = (1u << 4) | (type << 7) | (type << 10) | (1u << 16) | ((uint32_t)(HDP >> 3) << 17) | ((uint32_t)(PR_ROWS >> 4) << 24);
        auto scores = [&](int m, uint32_t k_tile) {  // the small products first
            const uint32_t d = tmem + m * 256 + C::S_COL, q = q_smem + m * PLANES * C::QBYTES;
            uint32_t add = 0;
#pragma unroll
            for (int part = PLANES == 2 ? 0 : 2; part < 3; part++) {
                const uint32_t qa = q + (part == 1 ? C::QBYTES : 0), ka = k_tile + (part == 0 ? C::KBYTES : 0);
#pragma unroll
                for (int ks = 0; ks < HDP / 16; ks++) {
                    umma_ss(d, umma_desc(qa + (ks / 4) * PR_ROWS * 128 + (ks % 4) * 32, 16), umma_desc(ka + (ks / 4) * NK * 128 + (ks % 4) * 32, 16), idesc_s, add);
                    add = 1;
                }
            }
        };
        auto weighted = [&](int m, int i, uint32_t v_tile) {
            const uint32_t d = tmem + m * 256 + C::O_COL + (C::O_BUFS == 2 ? (i & 1) * HDP : 0), p = tmem + m * 256 + C::S_COL;
            uint32_t add = C::O_IN_TMEM && i > 0;
#pragma unroll
            for (int part = PLANES == 2 ? 0 : 2; part < 3; part++) {
#pragma unroll
                for (int ks = 0; ks < NK / 16; ks++) {
                    // P of 32 keys: 16 columns, of f32 followed by the 16 of its low parts
                    const uint32_t pa = PLANES == 1 ? p + ks * 8 : p + (ks / 2) * 32 + (ks % 2) * 8 + (part == 1 ? 16 : 0);
                    umma_ts(d, pa, umma_desc(v_tile + (part == 0 ? C::KBYTES : 0) + ks * 2048, NK * 128), idesc_o, add);
                    add = 1;
                }
            }
        };
        bool ok = true;
        if (nt > 0) ok = bar_wait(bar, &bar->q_full, 0) && bar_wait(bar, &bar->full[0], 0);
        ok = __all_sync(0xffffffffu, ok);
        if (ok && nt > 0) {
            tc_fence_after();
            if (leader) {
                for (int m = 0; m < 2; m++)
                    if (n_tiles[m] > 0) {
                        scores(m, ring);
                        umma_commit(&bar->s_full[m]);
                    }
                umma_commit(&bar->empty[0]);
            }
            __syncwarp();
        }
        for (int i = 0; i < nt && ok; i++) {
            const int gv = 2 * i + 1, gk = gv + 1, sv = gv % NS, uv = gv / NS, sk = gk % NS, uk = gk / NS;
            ok = bar_wait(bar, &bar->ready[sv], ((NS & 1) ? uv >> 1 : uv) & 1);
            for (int m = 0; m < 2 && ok; m++) {
                if (i >= n_tiles[m]) continue;
                ok = bar_wait(bar, &bar->p_ready[m], i & 1);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                if (leader) weighted(m, i, ring + sv * C::SLOT);
                __syncwarp();
                if (i + 1 < n_tiles[m]) {
                    ok = __all_sync(0xffffffffu, bar_wait(bar, &bar->full[sk], uk & 1));
                    if (!ok) break;
                    tc_fence_after();
                    if (leader) scores(m, ring + sk * C::SLOT);
                }
                if (leader) umma_commit(&bar->s_full[m]);  // P V of this tile and S of the next
                __syncwarp();
            }
            ok = __all_sync(0xffffffffu, ok);
            if (ok && leader) {
                umma_commit(&bar->empty[sv]);
                if (i + 1 < nt) umma_commit(&bar->empty[sk]);
            }
            __syncwarp();
        }
    } else if (warp == 2) {
        // ── V check ──────────────────────────────────────────────────────────
        constexpr uint32_t EXP = std::is_same<T16, __nv_bfloat16>::value ? 0x7F807F80u : 0x7C007C00u;  // exponent bits, and
        constexpr uint32_t ONE = std::is_same<T16, __nv_bfloat16>::value ? 0x00800080u : 0x04000400u;  // their lowest one
        for (int i = 0; i < nt; i++) {
            const int g = 2 * i + 1, s = g % NS;
            if (!__all_sync(0xffffffffu, bar_wait(bar, &bar->full[s], (g / NS) & 1))) break;
            if (i >= first_masked) {
                uint8_t* tile = sm + 2 * PLANES * C::QBYTES + s * C::SLOT;
                uint32_t found[4] = {0, 0, 0, 0};
                for (int r = 0; r < NK; r += 4) {  // 8 lanes to a row of 128 bytes
                    bool odd = false;
#pragma unroll
                    for (int c = 0; c < PLANES * C::CH; c++) {
                        uint4* at = reinterpret_cast<uint4*>(tile + c * NK * 128 + (r + lane / 8) * 128) + lane % 8;
                        uint4 w = *at;
                        uint32_t* u = reinterpret_cast<uint32_t*>(&w);
                        uint32_t hit = 0;
#pragma unroll
                        for (int x = 0; x < 4; x++) hit |= (u[x] & EXP) + ONE;
                        if (hit & 0x80008000u) {
                            odd = true;
#pragma unroll
                            for (int x = 0; x < 4; x++) {
                                const uint32_t h = (u[x] & EXP) + ONE;
                                if (h & 0x8000u) u[x] &= 0xFFFF0000u;
                                if (h & 0x80000000u) u[x] &= 0x0000FFFFu;
                            }
                            *at = w;
                        }
                    }
                    const uint32_t votes = __ballot_sync(0xffffffffu, odd);
                    if (votes) {
                        uint32_t rows = 0;
#pragma unroll
                        for (int x = 0; x < 4; x++) rows |= ((votes >> (8 * x)) & 255u) ? 1u << x : 0u;
#pragma unroll
                        for (int x = 0; x < 4; x++)
                            if (r / 32 == x) found[x] |= rows << (r % 32);
                    }
                }
                if (lane < 4) bar->mask[i - first_masked][lane] = lane == 0 ? found[0] : lane == 1 ? found[1] : lane == 2 ? found[2] : found[3];
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) bar_arrive(&bar->checked[i - first_masked]);
            }
            __syncwarp();
            if (lane == 0) bar_arrive(&bar->ready[s]);
        }
    } else if (warp >= 4) {
        // ── softmax: one row per thread ──────────────────────────────────────
        const int m = (warp - 4) >> 2, r = (warp & 3) * 32 + lane, n = n_tiles[m];
        const int j = m * a.tile_tokens + r / a.group, head = kvh * a.group + r % a.group;
        const bool real = r < a.tile_tokens * a.group && j < blk.tokens;
        const int limit = real ? blk.visible(j) : 0;
        const uint32_t t_s = tmem + m * 256 + C::S_COL + ((uint32_t)((warp & 3) * 32) << 16), t_o = t_s + C::O_COL;
        const float NEG = __int_as_float(0xFF800000);
        float row_max = NEG, row_sum = 0.0f;
        float o[C::O_IN_TMEM ? 1 : HDP];
        bool ok = true;
        if constexpr (C::O_IN_TMEM) {
            for (int i = 0; i < n; i++) {
                if (!(ok = __all_sync(0xffffffffu, bar_wait(bar, &bar->s_full[m], i & 1)))) break;
                tc_fence_after();
                float s[NK];
#pragma unroll
                for (int c = 0; c < NK / 32; c++) tmem_ld32(t_s + 32 * c, s + 32 * c);
                tmem_ld_wait();
                const int seen = limit - i * NK;
                if (__any_sync(0xffffffffu, seen < NK)) {
#pragma unroll
                    for (int c = 0; c < NK; c++)
                        if (c >= seen) s[c] = NEG;
                }
                float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int c = 4; c < NK; c++) top[c & 3] = fmaxf(top[c & 3], s[c]);
                const float tile_max = __fmul_rn(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), a.scale_log2);
                const bool grown = tile_max > row_max + PR_LAZY || (row_max == NEG && tile_max > NEG);
                if (__any_sync(0xffffffffu, grown)) {
                    float f = 1.0f;
                    if (grown) {
                        f = exp2_approx(row_max - tile_max);
                        row_max = tile_max;
                        row_sum = __fmul_rn(row_sum, f);
                    }
                    if (i > 0) {
#pragma unroll 1
                        for (int c = 0; c < HDP; c += 32) {
                            float x[32];
                            tmem_ld32(t_o + c, x);
                            tmem_ld_wait();
#pragma unroll
                            for (int d = 0; d < 32; d++) x[d] = __fmul_rn(x[d], f);
                            tmem_st32(t_o + c, x);
                        }
                    }
                }
                const float base = row_max == NEG ? 0.0f : -row_max;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < NK / 32; c++) {
                    uint32_t p[16];
#pragma unroll
                    for (int x = 0; x < 16; x++) {
                        const float p0 = exp2_approx(fmaf(s[32 * c + 2 * x], a.scale_log2, base)), p1 = exp2_approx(fmaf(s[32 * c + 2 * x + 1], a.scale_log2, base));
                        sum[(2 * x) & 3] += p0, sum[(2 * x + 1) & 3] += p1;
                        p[x] = pack16<T16>(p0, p1);
                    }
                    tmem_st16(t_s + 16 * c, p);
                }
                row_sum += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(&bar->p_ready[m]);
            }
            if (n > 0 && ok) ok = __all_sync(0xffffffffu, bar_wait(bar, &bar->s_full[m], n & 1));
            tc_fence_after();
        } else {
#pragma unroll
            for (int d = 0; d < HDP; d++) o[d] = 0.0f;
            const float row_scale = real ? __fmul_rn(a.q_inv[(size_t)(blk.token0 + j) * a.p.n_heads + head], a.scale_log2) : 0.0f;
            const float* k_inv = a.k_inv + (size_t)key_slot0 * a.p.n_kv + kvh;
            const float* v_inv = a.v_inv + (size_t)key_slot0 * a.p.n_kv + kvh;
            float rescale = 0.0f;  // of what `o` holds, for the tile whose P V is still in tensor memory
            auto take_o = [&](int i) {
                const float f = v_inv[(size_t)i * a.p.n_kv];
#pragma unroll
                for (int c = 0; c < HDP; c += 32) {
                    float x[32];
                    tmem_ld32(t_o + (C::O_BUFS == 2 ? (i & 1) * HDP : 0) + c, x);
                    tmem_ld_wait();
#pragma unroll
                    for (int d = 0; d < 32; d++) o[c + d] = fmaf(x[d], f, __fmul_rn(o[c + d], rescale));
                }
            };
            for (int i = 0; i < n; i++) {
                const float scale = __fmul_rn(row_scale, k_inv[(size_t)i * a.p.n_kv]);
                if (!(ok = __all_sync(0xffffffffu, bar_wait(bar, &bar->s_full[m], i & 1)))) break;
                tc_fence_after();
                const int seen = limit - i * NK;
                const bool masked = __any_sync(0xffffffffu, seen < NK);
                float top = NEG;
#pragma unroll
                for (int c = 0; c < NK / 32; c++) {
                    float s[32];
                    tmem_ld32(t_s + 32 * c, s);
                    tmem_ld_wait();
                    if (masked) {
#pragma unroll
                        for (int x = 0; x < 32; x++)
                            if (32 * c + x >= seen) s[x] = NEG;
                    }
#pragma unroll
                    for (int x = 0; x < 32; x++) top = fmaxf(top, s[x]);
                }
                if (C::O_BUFS == 1 && i > 0) take_o(i - 1);
                const float new_max = fmaxf(row_max, __fmul_rn(top, scale));
                const float f = row_max == NEG ? 0.0f : exp2_approx(row_max - new_max);
                // weights up to 2^8, so that the low parts of small ones stay in f16's range
                const float base = new_max == NEG ? 0.0f : PR_LAZY - new_max;
                row_max = new_max;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < NK / 32; c++) {
                    float s[32];
                    tmem_ld32(t_s + 32 * c, s);
                    tmem_ld_wait();
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int x = 0; x < 32; x += 2) {
                        float p[2], h[2];
#pragma unroll
                        for (int y = 0; y < 2; y++) {
                            float v = fmaf(s[x + y], scale, base);
                            if (masked && 32 * c + x + y >= seen) v = NEG;
                            p[y] = exp2_approx(v);
                            h[y] = __uint_as_float(__float_as_uint(p[y]) & 0xFFFFE000u);  // 11 bits: exact in f16
                            sum[(x + y) & 3] += p[y];
                        }
                        hi[x / 2] = pack16<T16>(h[0], h[1]);
                        lo[x / 2] = pack16<T16>(__fsub_rn(p[0], h[0]), __fsub_rn(p[1], h[1]));
                    }
                    tmem_st16(t_s + 32 * c, hi);
                    tmem_st16(t_s + 32 * c + 16, lo);
                }
                row_sum = fmaf(row_sum, f, (sum[0] + sum[1]) + (sum[2] + sum[3]));
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(&bar->p_ready[m]);
                if (C::O_BUFS == 2 && i > 0) take_o(i - 1);
                rescale = f;
            }
            if (n > 0 && ok) ok = __all_sync(0xffffffffu, bar_wait(bar, &bar->s_full[m], n & 1));
            tc_fence_after();
            if (n > 0 && ok) take_o(n - 1);
        }
        for (int i = first_masked; i < nt && ok; i++) ok = __all_sync(0xffffffffu, bar_wait(bar, &bar->checked[i - first_masked], 0));

        // ── the rows: quotient, values that are not finite, rounding ─────────
        const float inv = limit > 0 ? __fdiv_rn(1.0f, row_sum) : 0.0f;
        T* out = reinterpret_cast<T*>(a.p.out) + ((size_t)(blk.token0 + j) * a.p.n_heads + head) * hd;
#pragma unroll
        for (int c = 0; c < HDP; c += 32) {
            float x[32];
            if (C::O_IN_TMEM) {
                if (n > 0) {  // (uniform in the warp)
                    tmem_ld32(t_o + c, x);
                    tmem_ld_wait();
                }
            } else {
#pragma unroll
                for (int d = 0; d < 32; d++) x[d] = o[C::O_IN_TMEM ? 0 : c + d];
            }
#pragma unroll
            for (int d = 0; d < 32; d++) x[d] = limit > 0 ? __fmul_rn(x[d], inv) : 0.0f;
            if (!ok) {
#pragma unroll
                for (int d = 0; d < 32; d++) x[d] = __int_as_float(0x7FC00000);
            }
            for (int i = first_masked; i < nt; i++)
                for (int w = 0; w < NK / 32; w++)
                    for (uint32_t bits = bar->mask[i - first_masked][w]; bits; bits &= bits - 1) {
                        const int t = i * NK + w * 32 + __ffs(bits) - 1;
                        if (t >= limit) continue;
                        const T* v = reinterpret_cast<const T*>(a.p.v) + (size_t)(blk.key0 + t) * a.p.v_stride + (size_t)kvh * hd;
#pragma unroll
                        for (int d = 0; d < 32; d++)
                            if (c + d < hd) {
                                const float y = to_f32(v[c + d]);
                                if (!(fabsf(y) <= 3.402823466e38f)) x[d] += y;
                            }
                    }
            if (real) {
                constexpr int V = 16 / (int)sizeof(T);
#pragma unroll
                for (int d = 0; d < 32; d += V)
                    if (c + d < hd) {
                        uint4 w;
                        if constexpr (sizeof(T) == 4)
                            w = make_uint4(__float_as_uint(x[d]), __float_as_uint(x[d + 1]), __float_as_uint(x[d + 2]), __float_as_uint(x[d + 3]));
                        else
                            w = make_uint4(pack16<T>(x[d], x[d + 1]), pack16<T>(x[d + 2], x[d + 3]), pack16<T>(x[d + 4], x[d + 5]), pack16<T>(x[d + 6], x[d + 7]));
                        *reinterpret_cast<uint4*>(out + c + d) = w;
                    }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        if (bar->abort)
            for (int i = 0; i < 64; i++) __nanosleep(1000);  // copies issued before the failure may still be landing
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// ── f32: two f16 parts and a power of two ───────────────────────────────────
// The power of two that takes a largest magnitude into [2^13, 2^14); 1 where there is none.
__device__ __forceinline__ float to_range(float top) {
    const int e = (int)((__float_as_uint(top) >> 23) & 255u);
    if (e == 0) return top > 0.0f ? 0x1p126f : 1.0f;  // (subnormal: as far as one factor goes)
    return __uint_as_float((uint32_t)min(253, 127 + 13 + 127 - e) << 23);
}
__device__ __forceinline__ void split4(float4 v, float f, uint2& hi, uint2& lo) {
    const float x[4] = {v.x, v.y, v.z, v.w};
    float h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float y = __fmul_rn(x[i], f);
        h[i] = __half2float(__float2half_rn(y));
        l[i] = fabsf(y) <= 65504.0f ? __fsub_rn(y, h[i]) : 0.0f;
    }
    hi = make_uint2(pack16<__half>(h[0], h[1]), pack16<__half>(h[2], h[3]));
    lo = make_uint2(pack16<__half>(l[0], l[1]), pack16<__half>(l[2], l[3]));
}
__device__ __forceinline__ float finite_abs(float x) { return fabsf(x) <= 3.402823466e38f ? fabsf(x) : 0.0f; }
__device__ __forceinline__ float finite_max(float4 v) { return fmaxf(fmaxf(finite_abs(v.x), finite_abs(v.y)), fmaxf(finite_abs(v.z), finite_abs(v.w))); }

struct SplitArgs {
    Prompts p;
    __half *q, *k, *v;  // [2][rows][heads * head_dim]
    float *q_inv, *k_inv, *v_inv;
    int tile, key_slots;  // keys of a tile; places for (sequence, tile)
};
constexpr int SP_THREADS = 256;

// CTAs [0, key_slots * n_kv * 2): a tile of K or V each; the others: rows of q, one (token, head) per warp.  Bound: HBM (4 bytes in, 4 out
// per element), the launch for short prompts.
__global__ void __launch_bounds__(SP_THREADS) k_split(const __grid_constant__ SplitArgs a) {
    pdl_trigger();
    pdl_wait();
    const int hd = a.p.head_dim, pieces = hd / 4, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles = a.key_slots * a.p.n_kv * 2;
    if ((int)blockIdx.x < tiles) {
        __shared__ float red[SP_THREADS / 32];
        const int val = blockIdx.x & 1, kvh = (blockIdx.x >> 1) % a.p.n_kv, slot = (blockIdx.x >> 1) / a.p.n_kv;
        const int32_t* ks = a.p.key_starts ? a.p.key_starts : a.p.starts;
        const int seq = find_seq(ks, a.p.n_seqs, a.p.n_keys, a.tile, slot);
        if (seq < 0) return;
        const int k0 = max(0, min(ks[seq], a.p.n_keys)), k1 = max(k0, min(ks[seq + 1], a.p.n_keys));
        const int first = k0 + (slot - (k0 / a.tile + seq)) * a.tile, rows = min(a.tile, k1 - first);
        if (rows <= 0) return;
        const float* src = (val ? (const float*)a.p.v + (size_t)first * a.p.v_stride : (const float*)a.p.k + (size_t)first * a.p.k_stride) + (size_t)kvh * hd;
        const size_t stride = val ? a.p.v_stride : a.p.k_stride, dim = (size_t)a.p.n_kv * hd, plane = (size_t)a.p.n_keys * dim;
        __half* dst = (val ? a.v : a.k) + (size_t)first * dim + (size_t)kvh * hd;
        float top = 0.0f;
        for (int i = threadIdx.x; i < rows * pieces; i += SP_THREADS) top = fmaxf(top, finite_max(reinterpret_cast<const float4*>(src + (i / pieces) * stride)[i % pieces]));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (lane == 0) red[warp] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < SP_THREADS / 32; w++) top = fmaxf(top, red[w]);
        const float f = to_range(top);
        for (int i = threadIdx.x; i < rows * pieces; i += SP_THREADS) {
            uint2 hi, lo;
            split4(reinterpret_cast<const float4*>(src + (i / pieces) * stride)[i % pieces], f, hi, lo);
            uint2* at = reinterpret_cast<uint2*>(dst + (i / pieces) * dim) + i % pieces;
            *at = hi;
            *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(at) + plane) = lo;
        }
        if (threadIdx.x == 0) (val ? a.v_inv : a.k_inv)[(size_t)slot * a.p.n_kv + kvh] = __fdiv_rn(1.0f, f);
        return;
    }
    const size_t at = (size_t)(blockIdx.x - tiles) * (SP_THREADS / 32) + warp, rows = (size_t)a.p.n_tokens * a.p.n_heads;
    if (at >= rows) return;
    const size_t token = at / a.p.n_heads, head = at % a.p.n_heads;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (lane < pieces) v = reinterpret_cast<const float4*>((const float*)a.p.q + token * a.p.q_stride + head * hd)[lane];
    float top = finite_max(v);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float f = to_range(top);
    uint2 hi, lo;
    split4(v, f, hi, lo);
    if (lane < pieces) {
        uint2* dst = reinterpret_cast<uint2*>(a.q + at * hd) + lane;
        *dst = hi;
        *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(dst) + rows * hd) = lo;
    }
    if (lane == 0) a.q_inv[at] = __fdiv_rn(1.0f, f);
}

// ── host side ───────────────────────────────────────────────────────────────
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled_fn() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) == cudaSuccess && found == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
    });
    return fn;
}
// 16-bit rows [planes][rows][heads][head_dim]; box: 64 columns (zeros behind head_dim) x box_heads x box_rows, 128-byte swizzle.
cudaError_t encode_heads(const void* base, bool bf16, int hd, int heads, int rows, int planes, size_t stride, int box_heads, int box_rows, CUtensorMap* out) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return cudaErrorNotSupported;
    const cuuint64_t dims[4] = {(cuuint64_t)hd, (cuuint64_t)heads, (cuuint64_t)rows, (cuuint64_t)planes};
    const cuuint64_t strides[3] = {(cuuint64_t)hd * 2, (cuuint64_t)stride * 2, (cuuint64_t)stride * 2 * (cuuint64_t)rows};
    const cuuint32_t box[4] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows, 1}, step[4] = {1, 1, 1, 1};
    const CUresult r = fn(out, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides, box,
                          step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

constexpr size_t up128(size_t n) { return (n + 127) & ~(size_t)127; }
int keys_per_tile(const Prompts& p) { return p.dtype == DT_F32 && p.head_dim > 64 ? Cfg<2, 128>::NK : Cfg<1, 64>::NK; }
int places(int rows, int seqs, int block) { return rows / block + seqs + 1; }

struct Workspace {
    size_t q, k, v, q_inv, k_inv, v_inv, bytes;
    explicit Workspace(const Prompts& p) {
        const size_t key_slots = (size_t)places(p.n_keys, p.n_seqs, keys_per_tile(p));
        size_t at = 0;
        auto take = [&at](size_t n) {
            const size_t here = at;
            at += up128(n);
            return here;
        };
        q = take((size_t)p.n_tokens * p.n_heads * p.head_dim * 4);
        k = take((size_t)p.n_keys * p.n_kv * p.head_dim * 4);
        v = take((size_t)p.n_keys * p.n_kv * p.head_dim * 4);
        q_inv = take((size_t)p.n_tokens * p.n_heads * 4);
        k_inv = take(key_slots * p.n_kv * 4);
        v_inv = take(key_slots * p.n_kv * 4);
        bytes = at;
    }
};

template <class T, int PLANES, int HDP>
cudaError_t launch_typed(cudaStream_t st, const Prompts& p, void* workspace) {
    using C = Cfg<PLANES, HDP>;
    static RaisedPerDevice limit;
    cudaError_t e = raise_dynamic_smem(limit, (const void*)k_attention_prompts<T, PLANES, HDP>, C::SMEM);
    if (e != cudaSuccess) return e;
    PromptArgs a{};
    a.p = p;
    a.group = p.n_heads / p.n_kv;
    a.tile_tokens = PR_ROWS / a.group;
    a.slots = places(p.n_tokens, p.n_seqs, 2 * a.tile_tokens);
    a.zero_rest = p.zero_rest;
    a.scale_log2 = 1.4426950408889634f / sqrtf((float)p.head_dim);
    const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
    const void *q = p.q, *k = p.k, *v = p.v;
    size_t qs = p.q_stride, ks = p.k_stride, vs = p.v_stride;
    if (PLANES == 2) {
        const Workspace w(p);
        uint8_t* base = static_cast<uint8_t*>(workspace);
        SplitArgs s{p, (__half*)(base + w.q), (__half*)(base + w.k), (__half*)(base + w.v), (float*)(base + w.q_inv), (float*)(base + w.k_inv),
                    (float*)(base + w.v_inv), C::NK, p.n_keys > 0 ? places(p.n_keys, p.n_seqs, C::NK) : 0};
        const long long ctas = (long long)s.key_slots * p.n_kv * 2 + ((long long)p.n_tokens * p.n_heads + SP_THREADS / 32 - 1) / (SP_THREADS / 32);
        if (ctas > 0x7FFFFFFFll) return cudaErrorInvalidValue;
        g_kernel_launches++;
        if ((e = launch_pdl(st, k_split, dim3((unsigned)ctas), dim3(SP_THREADS), 0, s)) != cudaSuccess) return e;
        q = s.q, k = s.k, v = s.v;
        qs = (size_t)p.n_heads * p.head_dim, ks = vs = (size_t)p.n_kv * p.head_dim;
        a.q_inv = s.q_inv, a.k_inv = s.k_inv, a.v_inv = s.v_inv;
    }
    CUtensorMap mq, mk, mv;
    if ((e = encode_heads(q, bf16, p.head_dim, p.n_heads, p.n_tokens, PLANES, qs, a.group, a.tile_tokens, &mq)) != cudaSuccess) return e;
    mk = mv = mq;  // (without any keys: never read)
    if (p.n_keys > 0) {
        if ((e = encode_heads(k, bf16, p.head_dim, p.n_kv, p.n_keys, PLANES, ks, 1, C::NK, &mk)) != cudaSuccess) return e;
        if ((e = encode_heads(v, bf16, p.head_dim, p.n_kv, p.n_keys, PLANES, vs, 1, C::NK, &mv)) != cudaSuccess) return e;
    }
    const long long grid = (long long)a.slots * p.n_kv + (p.zero_rest ? PR_ZERO_CTAS : 0);
    if (grid > 0x7FFFFFFFll) return cudaErrorInvalidValue;
    g_kernel_launches++;
    return launch_pdl(st, k_attention_prompts<T, PLANES, HDP>, dim3((unsigned)grid), dim3(PR_THREADS), C::SMEM, mq, mk, mv, a);
}

}  // namespace

size_t attention_prompts_workspace(const Prompts& p) { return p.dtype == DT_F32 ? Workspace(p).bytes : 0; }

cudaError_t launch_attention_prompts(cudaStream_t st, const Prompts& p, void* workspace) {
    const bool wide = p.head_dim > 64;
    if (p.dtype == DT_F32) return wide ? launch_typed<float, 2, 128>(st, p, workspace) : launch_typed<float, 2, 64>(st, p, workspace);
    if (p.dtype == DT_F16) return wide ? launch_typed<__half, 1, 128>(st, p, workspace) : launch_typed<__half, 1, 64>(st, p, workspace);
    return wide ? launch_typed<__nv_bfloat16, 1, 128>(st, p, workspace) : launch_typed<__nv_bfloat16, 1, 64>(st, p, workspace);
}

}  // namespace wick

// Causal attention of packed prompts with grouped heads on tcgen05.
//
// Token j of a sequence with nq tokens and nk keys attends its keys t <= j + nk - nq:  o_j = sum_t p_t v_t / sum_t p_t with
// p_t = 2^(x_t - m), x_t = log2(e) / sqrt(d) q_j . k_t, m a running maximum.
//
// A CTA per SM walks over items: 2 x 128 rows of one KV head.  A row is a (token, query head of the group) pair, 128 / group tokens to a row tile, so
// that a K / V tile that lies in shared memory serves every head of its group and short prompts fill the rows.  K and V tiles of NK keys go through
// one ring of TMA slots (K0 V0 K1 V1 ..), which runs on from item to item.  Per row tile: S = Q K^T (tcgen05, S in tensor memory) -> the tile's four
// softmax warps, one row per thread -> P in tensor memory -> P V with P as the A operand from there.  The two row tiles alternate: while one is
// in the tensor core the other is in its softmax; and an item's last rows are written while the next one's first scores are computed.
//
// f16, bf16: one product each; O stays in tensor memory, and is rescaled only where a row's maximum has grown by more than 2^8 (a weight is at most
//   2^8 then, times 2^7 in f16 and 2^-8 in bf16; the last maximum that was used cancels in the quotient).  Weights are rounded to the operands' type, half a step
//   each, as the tensor core takes them; their sum is of the unrounded ones.  The tensor core adds with truncation: O is taken out and added up in
//   f32 every 64 tiles (8192 keys: 5e-5 of the sum; 131072 without this were 7e-4, 1.5 half steps of f16).
// f32: every operand is split into two f16 parts, x = 2^e (hi + lo), 22 bits, with one power of two per row of Q and per tile of K and V (K and V by
//   k_split; a row of Q where it lies in shared memory, by the thread that owns it), and a product is hi hi + hi lo + lo hi (lo lo is 2^-22 of it).
//   O is taken out after every tile and added up in registers, as with truncated additions a sum over thousands of keys would drift by 1e-5.
//   An element is held to 2^-22 of itself or 2^-24 of its row's largest.  Rows of a K or V tile that are too far apart for one power of two (a row's
//   largest element below 2^-14 of the others', or above them) are zeros in the parts: the threads that attend such a far key compute its score, and
//   add its weighted value, in f32 from K and V themselves (eight prompts of 1000 tokens, 32 / 8 heads of 64: 161 us without far keys, 323 with one in
//   every tile, 1075 with one in 16).  What a token does not attend does not change its result beyond that rounding.  Keys with infinities or NaN are
//   far, too; values that are not finite are zeros in the parts and are added to the rows that attend them at the end.
//
// Few items with many keys (a chunk of tokens behind a long prefix): the keys of an item are cut into `splits` parts, each an item of its own,
// whose sums go to the workspace in f32 and are joined by k_join.
//
// Masked places may hold anything.  Scores are masked after the product; V is different, 0 * NaN is NaN: a warp looks at every V
// tile that some row sees in part, zeroes what is not finite (in f32: left behind the sequences in the workspace), and notes the keys; rows that
// attend such a key add its values at the end.
//
// Bound, on a B200: the softmax and its MMAs in turn, two softmax warps to a scheduler, which wait for one another's results more than they issue (issue
// slots 40 % in f32, 33 % in 16 bits).  A pair of tiles, one of each row tile, takes (slope of the time over the keys, 1965 MHz) in f32 5600 cycles (heads
// of 64, 128 keys; 54 % of them MMAs by count) or 5700 (heads of 128, 64 keys), in 16 bits 3600 to 3900 (the special function unit needs 2048 for its
// exponentials, the MMAs 1024 with heads of 64 and 2048 with 128).  Eight prompts of 250 to 1001 tokens, 32 / 8 heads of 64, f32: 97 us (tensor pipe
// 35 %); one of 8000, heads of 128, bf16: 451 us (1160 TFLOP/s; tensor pipe 54 %, special function unit 54 %), 521 under the power cap.  Loops that
// run once per item stay rolled: unrolled they took longer to fetch than to run (161 -> 116 us in the first case, before other steps).
//
// Every wait is bounded: on expiry all roles leave their loops and all rows of the CTA's items become NaN.
#include <cuda.h>
#include <algorithm>
#include <cmath>
#include <mutex>

#include "serving.cuh"

namespace wick {

namespace {

constexpr int PR_ROWS = 128;      // rows of a tile == lanes of tensor memory
constexpr int PR_THREADS = 384;   // TMA, MMA, V check, items; 2 x 4 softmax warps
constexpr int PR_ITEMS = 3;       // items that are known ahead
constexpr int PR_MASKED = 8;      // tiles that some row of a CTA sees in part: at most 256 / 64 + 2
constexpr int PR_CARRY = 64;     // tiles
constexpr float PR_LAZY = 8.0f, PR_DOWN = 0x1p-8f;  // 2^-PR_LAZY

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
    // columns of a row tile's 256: S, O, and P over S or, where there is room, beside it (the next S need not wait for P V then)
    static constexpr bool P_APART = PLANES == 1 && HDP == 64;
    static constexpr int S_COL = 0, P_COL = P_APART ? NK : 0, O_COL = NK + (P_APART ? NK / 2 : 0);
    static_assert(O_COL + O_BUFS * HDP <= 256 && NS >= 3, "tensor or shared memory");
    static constexpr size_t SMEM = 1024 + (size_t)2 * PLANES * QBYTES + (size_t)NS * SLOT + 1024;
};

constexpr int FAR_WORDS = 4;  // of 32 rows; a tile has at most 128

struct Item {
    int token0, tokens;   // first token (a row of q), tokens
    int key0, keys;       // first key (a row of k), keys of the sequence
    int first_visible;    // keys that the first token attends (may be negative)
    int key_slot0, kvh;   // place of the sequence's first key tile; KV head (-1: no more items)
    int part;             // of the block's keys
    int n_tiles[2];       // tiles of keys that the two row tiles see
    uint32_t mask[PR_MASKED][4];  // keys of the tiles from first_masked() on whose values are not finite
    __device__ __forceinline__ int visible(int j) const { return max(0, min(first_visible + j, keys)); }
    __device__ __forceinline__ int nt() const { return max(n_tiles[0], n_tiles[1]); }
    template <int NK>
    __device__ __forceinline__ int first_masked() const { return max(0, first_visible) / NK; }  // tiles from here on are seen in part by some row
};
struct Shared {
    unsigned long long q_full[2], q_raw[2], q_empty, k_full[6], v_full[6], empty[6], ready[6], s_full[2], s_read[2], p_ready[2], o_full[2];
    unsigned long long item_full[PR_ITEMS], item_empty[PR_ITEMS], checked[PR_ITEMS];
    Item item[PR_ITEMS];
    uint32_t tmem_base, wait_rounds;
    volatile uint32_t abort;
};
static_assert(sizeof(Shared) <= 1024, "room behind the ring");

// What the kernels read besides the tensor maps.
struct PromptArgs {
    Prompts p;
    const float *k_inv, *v_inv;          // f32: the powers of two taken out of K / V tiles, negative where the tile has far or bad rows,
    const uint32_t *k_far, *v_far;       // and, for those tiles, which: bit per row, [slot][n_kv][FAR_WORDS];
    const uint32_t* v_bad;               // rows of V with elements that are not finite, likewise
    int group, tile_tokens;              // query heads per KV head, tokens of a row tile
    int slots;                           // places for (sequence, block of 2 * tile_tokens tokens)
    int splits;                          // parts of a block's keys, and where their rows' sums go: [splits][tokens][heads][head_dim], [..][2]
    float *part_o, *part_ml;
    int zero_rest;
    int wide_rows;                       // rows of out start on 32-byte boundaries
    float scale_log2;
    ServingWaits waits;
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
// false: the limit, or another role has given up
__device__ __forceinline__ bool bar_wait(Shared* b, void* bar, uint32_t parity) {
    for (uint32_t i = 1;; i++) {
        if (mbar_try_wait(smem_u32(bar), parity)) return true;
        if ((i & 255u) == 0) {
            if (b->abort) return false;
            if (i >= b->wait_rounds) break;
        }
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
__device__ __forceinline__ float tmem_ld1(uint32_t addr) {
    float r;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=f"(r) : "r"(addr) : "memory");
    return r;
}
__device__ __forceinline__ void tmem_st1(uint32_t addr, float v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Shared memory by 32-bit address (the aligned buffer's pointer is a generic one to the compiler)
__device__ __forceinline__ void lds_4(uint32_t at, float* v) {
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void sts_4(uint32_t at, const uint32_t* v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
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

// ── f32: two f16 parts and a power of two ───────────────────────────────────
// The power of two that takes a largest magnitude into [2^13, 2^14); 1 where there is none.
__device__ __forceinline__ float to_range(float top) {
    const int e = (int)((__float_as_uint(top) >> 23) & 255u);
    if (e == 0) return top > 0.0f ? 0x1p126f : 1.0f;  // (subnormal: as far as one factor goes)
    return __uint_as_float((uint32_t)min(253, 127 + 13 + 127 - e) << 23);
}
__device__ __forceinline__ void split4(float4 v, float f, uint2& hi, uint2& lo) {  // (finite, and below 2^14 with the factor)
    const float x[4] = {v.x, v.y, v.z, v.w};
    float h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float y = __fmul_rn(x[i], f);
        h[i] = __uint_as_float(__float_as_uint(y) & 0xFFFFE000u);  // 11 bits: exact in f16
        l[i] = __fsub_rn(y, h[i]);
    }
    hi = make_uint2(pack16<__half>(h[0], h[1]), pack16<__half>(h[2], h[3]));
    lo = make_uint2(pack16<__half>(l[0], l[1]), pack16<__half>(l[2], l[3]));
}
constexpr float MAX_F32 = 3.402823466e38f;
__device__ __forceinline__ float finite(float x) { return fabsf(x) <= MAX_F32 ? x : 0.0f; }
__device__ __forceinline__ float4 finite(float4 v) { return make_float4(finite(v.x), finite(v.y), finite(v.z), finite(v.w)); }
__device__ __forceinline__ uint32_t magnitude(float4 v) {  // the largest one's bits
    return max(max(__float_as_uint(v.x) & 0x7FFFFFFFu, __float_as_uint(v.y) & 0x7FFFFFFFu), max(__float_as_uint(v.z) & 0x7FFFFFFFu, __float_as_uint(v.w) & 0x7FFFFFFFu));
}

// The blocks of 2 * tile_tokens tokens, counted through the sequences, by a whole warp: how many there are (want < 0), or which sequence has number
// `want` and which of its blocks that is (*seq -1: none).  From PR_WALK sequences on, numbers are places as of find_seq, not all of which
// have a block: two or three steps in place of a walk over 32 sequences at a time, but items dealt less evenly.  (Prompts of 64 tokens, 16 / 8 heads of 64, f16: 33,
// 128, 256, 512, 1024 sequences walked through 15, 40, 75, 156, 421 us, searched for 19, 42, 70, 132, 257; of 200 tokens 31, 100, 192, 378, 936 and 37,
// 103, 190, 366, 705.)
constexpr int PR_WALK = 256;
__device__ __forceinline__ int count_blocks(const PromptArgs& a, int want, int* seq, int* at) {
    const int block = 2 * a.tile_tokens, lane = threadIdx.x & 31;
    *seq = -1, *at = 0;
    if (a.p.n_seqs > PR_WALK) {
        if (want < 0) return a.slots;
        *seq = find_seq(a.p.starts, a.p.n_seqs, a.p.n_tokens, block, want);
        if (*seq >= 0) *at = want - (max(0, min(a.p.starts[*seq], a.p.n_tokens)) / block + *seq);
        return a.slots;
    }
    int before = 0;
    for (int s0 = 0; s0 < a.p.n_seqs; s0 += 32) {
        const int s = s0 + lane;
        int n = 0;
        if (s < a.p.n_seqs) {
            const int q0 = max(0, min(a.p.starts[s], a.p.n_tokens)), q1 = max(q0, min(a.p.starts[s + 1], a.p.n_tokens));
            n = (q1 - q0 + block - 1) / block;
        }
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, want >= 0 && before + upto > want);
        if (past) {
            const int l = __ffs(past) - 1;
            *seq = s0 + l;
            *at = want - before - __shfl_sync(0xffffffffu, upto - n, l);
            return 0;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return before;
}

// Block blk of a sequence, with all its keys; false: there is none.
template <int NK>
__device__ __forceinline__ bool block_of(const PromptArgs& a, int seq, int blk, Item& it) {
    const int block = 2 * a.tile_tokens;
    if (seq < 0) return false;
    const int32_t* ks = a.p.key_starts ? a.p.key_starts : a.p.starts;
    const int s0 = a.p.starts[seq], s1 = a.p.starts[seq + 1], t0 = ks[seq], t1 = ks[seq + 1];
    const int q0 = max(0, min(s0, a.p.n_tokens)), q1 = max(q0, min(s1, a.p.n_tokens));
    const int k0 = max(0, min(t0, a.p.n_keys)), k1 = max(k0, min(t1, a.p.n_keys));
    const int at = blk * block;
    if (at >= q1 - q0) return false;
    it.token0 = q0 + at;
    it.tokens = min(block, q1 - it.token0);
    it.key0 = k0, it.keys = k1 - k0;
    it.first_visible = at + 1 + it.keys - (q1 - q0);
    it.key_slot0 = k0 / NK + seq;
#pragma unroll
    for (int m = 0; m < 2; m++) {
        const int rows = min(a.tile_tokens, it.tokens - m * a.tile_tokens);
        it.n_tiles[m] = rows > 0 ? (it.visible(m * a.tile_tokens + rows - 1) + NK - 1) / NK : 0;
    }
    return true;
}
// Where part `part` of nt tiles begins: equal parts (one may be empty: an item without tiles).
__device__ __forceinline__ int part_begin(int nt, int part, int splits) { return (int)((long long)nt * part / splits); }
// A part of a block's keys as an item (one without tiles too: its rows' maxima of -inf tell the join).
template <int NK>
__device__ __forceinline__ void part_of(const PromptArgs& a, int kvh, int part, Item& it) {
    it.kvh = kvh;
    it.part = part;
    if (a.splits > 1) {  // the sequence as this part sees it: its keys begin at the part's first tile
        const int nt = it.nt(), t0 = part_begin(nt, part, a.splits), t1 = part_begin(nt, part + 1, a.splits);
        it.key0 += t0 * NK, it.keys -= t0 * NK, it.first_visible -= t0 * NK, it.key_slot0 += t0;
#pragma unroll
        for (int m = 0; m < 2; m++) it.n_tiles[m] = max(0, min(it.n_tiles[m], t1) - t0);
    }
}

// The same value, from which nothing is computed ahead: what only far keys need takes no registers of the loops around.
template <class X>
__device__ __forceinline__ X aside(X x) {
    if constexpr (sizeof(X) == 8)
        asm volatile("" : "+l"(x));
    else
        asm volatile("" : "+r"(x));
    return x;
}
__device__ __forceinline__ size_t far_tile(const PromptArgs& a, const Item* it, int i) {
    return ((size_t)(it->key_slot0 + i) * a.p.n_kv + it->kvh) * FAR_WORDS;
}

// Scores so large that their distance from the maximum, as one product and sum that is rounded once, would see the rounding of the maximum itself: half a
// unit of it must stay well below 1.  From there on a score is rounded before the maximum is taken off.
__device__ __forceinline__ bool coarse(float top) { return fabsf(top) > 0x1p22f && top > __int_as_float(0xFF800000); }

// A CTA's items one after the other, by a whole warp: the list is dealt to the CTAs forwards and backwards in turn, and begins with the
// blocks that have the most keys, so that the CTAs end about together.  Up to 32 sequences (a lane each) their last blocks come first, then
// their last but one ..; with more, one sequence's blocks after the other's, backwards.
template <int NK>
struct Deal {
    int blocks, mine, turn, level, above;  // blocks in all; this lane's sequence's; rounds so far; blocks of higher number than `level`
    bool by_level;
    __device__ __forceinline__ explicit Deal(const PromptArgs& a) : mine(0), turn(0), level(0), above(0), by_level(a.p.n_seqs <= 32) {
        int seq, blk;
        blocks = count_blocks(a, -1, &seq, &blk);
        if (by_level) {
            const int s = threadIdx.x & 31, block = 2 * a.tile_tokens;
            if (s < a.p.n_seqs) {
                const int q0 = max(0, min(a.p.starts[s], a.p.n_tokens)), q1 = max(q0, min(a.p.starts[s + 1], a.p.n_tokens));
                mine = (q1 - q0 + block - 1) / block;
            }
            level = __reduce_max_sync(0xffffffffu, mine) - 1;
        }
    }
    // false: the CTA has had its items
    __device__ __forceinline__ bool next(const PromptArgs& a, Item& it) {
        const int total = blocks * a.p.n_kv * a.splits;
        while (true) {
            const long long idx = (long long)turn * gridDim.x + ((turn & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
            if ((long long)turn * gridDim.x >= total) return false;
            turn++;
            if (idx >= total) continue;
            const int part = (int)idx % a.splits, place = (int)idx / a.splits, kvh = place % a.p.n_kv, number = place / a.p.n_kv;
            int seq = -1, blk = 0;
            if (by_level) {
                uint32_t have = __ballot_sync(0xffffffffu, mine > level);
                while (level > 0 && above + __popc(have) <= number) {
                    above += __popc(have);
                    level--;
                    have = __ballot_sync(0xffffffffu, mine > level);
                }
                const int lane = threadIdx.x & 31;
                const bool it_is = (have >> lane & 1) && __popc(have & ((1u << lane) - 1)) == number - above;
                seq = __ffs(__ballot_sync(0xffffffffu, it_is)) - 1, blk = level;
            } else {
                count_blocks(a, blocks - 1 - number, &seq, &blk);
            }
            if (block_of<NK>(a, seq, blk, it)) {
                part_of<NK>(a, kvh, part, it);
                return true;
            }
        }
    }
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
    Shared* sh = reinterpret_cast<Shared*>(sm + 2 * PLANES * C::QBYTES + NS * C::SLOT);
    const uint32_t q_smem = smem_u32(sm), ring = q_smem + 2 * PLANES * C::QBYTES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hd = a.p.head_dim;

    if (threadIdx.x == 0) {
        for (int m = 0; m < 2; m++) {
            bar_init(&sh->q_full[m], PLANES == 2 ? 4 : 1), bar_init(&sh->q_raw[m], 1);
            bar_init(&sh->s_full[m], 1), bar_init(&sh->s_read[m], 4), bar_init(&sh->p_ready[m], 4), bar_init(&sh->o_full[m], 1);
        }
        bar_init(&sh->q_empty, 1);
        for (int s = 0; s < NS; s++) bar_init(&sh->k_full[s], 1), bar_init(&sh->v_full[s], 1 + a.waits.missing), bar_init(&sh->empty[s], 1), bar_init(&sh->ready[s], 1);
        for (int i = 0; i < PR_ITEMS; i++) bar_init(&sh->item_full[i], 1), bar_init(&sh->item_empty[i], 11), bar_init(&sh->checked[i], 1);
        sh->abort = 0, sh->wait_rounds = a.waits.rounds;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh->tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_trigger();
    pdl_wait();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh->tmem_base;

    // Ring positions g = 0, 1, .. hold K0 V0 K1 V1 ..; K and V have barriers of their own, so that who waits for V needs nothing of the K's that share
    // its slot: an odd number of slots has them in turn, and a use's number among those of its kind is half its number then.
    auto use_parity = [](uint32_t g) { return ((NS & 1) ? g / NS >> 1 : g / NS) & 1; };
    // An item of the list, for a role: waits until it is known.  false: no more items (or a wait ran out).
    auto next_item = [&](uint32_t k) -> const Item* {
        if (!__all_sync(0xffffffffu, bar_wait(sh, &sh->item_full[k % PR_ITEMS], (k / PR_ITEMS) & 1))) return nullptr;
        const Item* it = &sh->item[k % PR_ITEMS];
        return it->kvh < 0 ? nullptr : it;
    };
    auto leave_item = [&](uint32_t k) {
        __syncwarp();
        if (lane == 0) bar_arrive(&sh->item_empty[k % PR_ITEMS]);
    };

    // Registers: the launch has 12 warps of 168; four give up 80 each, eight take 40 more (4 x 88 + 8 x 208 = 12 x 168).  One instruction for the
    // four, in front of their branches: a warpgroup executes it together.
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 3) {
            // ── items ────────────────────────────────────────────────────────────
            Deal<NK> deal(a);
            uint32_t k = 0;
            while (true) {
                Item it;
                if (!deal.next(a, it)) it.kvh = -1;
                if (!__all_sync(0xffffffffu, bar_wait(sh, &sh->item_empty[k % PR_ITEMS], ((k / PR_ITEMS) & 1) ^ 1))) break;
                if (lane == 0) {
                    Item* to = &sh->item[k % PR_ITEMS];
                    to->token0 = it.token0, to->tokens = it.tokens, to->key0 = it.key0, to->keys = it.keys, to->first_visible = it.first_visible;
                    to->key_slot0 = it.key_slot0, to->kvh = it.kvh, to->part = it.part, to->n_tiles[0] = it.n_tiles[0], to->n_tiles[1] = it.n_tiles[1];
                    bar_arrive(&sh->item_full[k % PR_ITEMS]);
                }
                __syncwarp();
                k++;
                if (it.kvh < 0) break;
            }
            if (a.zero_rest) {  // rows of no sequence
                const int first = max(0, min(a.p.starts[0], a.p.n_tokens)), last = max(first, min(a.p.starts[a.p.n_seqs], a.p.n_tokens));
                const size_t row = (size_t)a.p.n_heads * hd * sizeof(T) / 16, n = (size_t)(a.p.n_tokens - last + first) * row;
                for (size_t i = (size_t)blockIdx.x * 32 + lane; i < n; i += (size_t)gridDim.x * 32)
                    reinterpret_cast<uint4*>(a.p.out)[i < first * row ? i : i + (size_t)(last - first) * row] = make_uint4(0, 0, 0, 0);
            }
        } else if (warp == 0) {
            // ── TMA ──────────────────────────────────────────────────────────────
            uint32_t g = 0, qn = 0;  // ring positions; items with keys
            bool ok = true;
            for (uint32_t k = 0; ok; k++) {
                const Item* it = next_item(k);
                if (!it) break;
                const int nt = it->nt();
                if (nt > 0) {
                    if (lane == 0) {
                        // Q: 128-byte columns, 64 elements of 16 bits or 32 of f32 (which its owners turn into two parts where they lie)
                        constexpr int COLS = PLANES * C::CH, WIDTH = 64 / PLANES;
                        ok = bar_wait(sh, &sh->q_empty, (qn & 1) ^ 1);
                        for (int m = 0; m < 2 && ok; m++) {
                            if (it->n_tiles[m] == 0) continue;
                            unsigned long long* bar = PLANES == 2 ? &sh->q_raw[m] : &sh->q_full[m];
                            bar_expect(bar, (uint32_t)(COLS * a.group * a.tile_tokens * 128));
                            for (int c = 0; c < COLS; c++)
                                tma_4d(q_smem + m * PLANES * C::QBYTES + c * PR_ROWS * 128, &map_q, bar, c * WIDTH, it->kvh * a.group,
                                       it->token0 + m * a.tile_tokens, 0);
                        }
                        for (int i = 0; i < 2 * nt && ok; i++) {
                            const uint32_t s = (g + i) % NS, u = (g + i) / NS;
                            ok = bar_wait(sh, &sh->empty[s], (u & 1) ^ 1);
                            if (!ok) break;
                            unsigned long long* bar = (i & 1) ? &sh->v_full[s] : &sh->k_full[s];
                            bar_expect(bar, C::SLOT);
                            for (int p = 0; p < PLANES; p++)
                                for (int c = 0; c < C::CH; c++)
                                    tma_4d(ring + s * C::SLOT + p * C::KBYTES + c * NK * 128, (i & 1) ? &map_v : &map_k, bar, c * 64, it->kvh,
                                           it->key0 + (i >> 1) * NK, p);
                        }
                    }
                    ok = __all_sync(0xffffffffu, ok);
                    g += 2 * nt, qn++;
                }
                leave_item(k);
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
                    const uint32_t ka = k_tile + (part == 0 ? C::KBYTES : 0);
#pragma unroll
                    for (int ks = 0; ks < HDP / 16; ks++) {
                        // Q: 64 elements to a 128-byte column; of f32 32, the low parts behind the high ones
                        const uint32_t qa = PLANES == 1 ? q + (ks / 4) * PR_ROWS * 128 + (ks % 4) * 32
                                                        : q + (ks / 2) * PR_ROWS * 128 + (part == 1 ? 64 : 0) + (ks % 2) * 32;
                        umma_ss(d, umma_desc(qa, 16), umma_desc(ka + (ks / 4) * NK * 128 + (ks % 4) * 32, 16), idesc_s, add);
                        add = 1;
                    }
                }
            };
            auto weighted = [&](int m, int i, uint32_t buf, uint32_t v_tile) {
                const uint32_t d = tmem + m * 256 + C::O_COL + (C::O_BUFS == 2 ? buf * HDP : 0), p = tmem + m * 256 + C::P_COL;
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
            uint32_t g = 0, done[2] = {0, 0}, qn[2] = {0, 0};  // ring positions; tiles and items of each row tile so far
            bool ok = true;
            for (uint32_t k = 0; ok; k++) {
                const Item* it = next_item(k);
                if (!it) break;
                const int n0 = it->n_tiles[0], n1 = it->n_tiles[1], nt = max(n0, n1);
                // S of tile i of a row tile, in whose place (P_APART: behind whose reading) the one before has been
                auto issue_scores = [&](int m, uint32_t slot, int i) -> bool {
                    if (C::P_APART && done[m] + i > 0 && !__all_sync(0xffffffffu, bar_wait(sh, &sh->s_read[m], (done[m] + i - 1) & 1))) return false;
                    tc_fence_after();
                    if (leader) {
                        scores(m, ring + slot * C::SLOT);
                        umma_commit(&sh->s_full[m]);
                    }
                    __syncwarp();
                    return true;
                };
                if (nt > 0) {
                    ok = __all_sync(0xffffffffu, bar_wait(sh, &sh->k_full[g % NS], use_parity(g)));
                    for (int m = 0; m < 2 && ok; m++)
                        if (it->n_tiles[m] > 0) {
                            ok = __all_sync(0xffffffffu, bar_wait(sh, &sh->q_full[m], qn[m] & 1));
                            if (ok) ok = issue_scores(m, g % NS, 0);
                            qn[m]++;
                        }
                    if (ok && leader) {
                        umma_commit(&sh->empty[g % NS]);
                        if (nt == 1) umma_commit(&sh->q_empty);
                    }
                    __syncwarp();
                }
                for (int i = 0; i < nt && ok; i++) {
                    const uint32_t gv = g + 2 * i + 1, gk = gv + 1, sv = gv % NS, sk = gk % NS;
                    const bool more = i + 1 < nt;
                    if (C::P_APART && more) {  // the next scores first
                        ok = __all_sync(0xffffffffu, bar_wait(sh, &sh->k_full[sk], use_parity(gk)));
                        for (int m = 0; m < 2 && ok; m++)
                            if (i + 1 < it->n_tiles[m]) ok = issue_scores(m, sk, i + 1);
                        if (!ok) break;
                        if (leader) {
                            umma_commit(&sh->empty[sk]);
                            if (i + 2 == nt) umma_commit(&sh->q_empty);
                        }
                        __syncwarp();
                    }
                    ok = __all_sync(0xffffffffu, bar_wait(sh, &sh->ready[sv], use_parity(gv)));
                    for (int m = 0; m < 2 && ok; m++) {
                        const int n = m ? n1 : n0;
                        if (i >= n) continue;
                        ok = __all_sync(0xffffffffu, bar_wait(sh, &sh->p_ready[m], (done[m] + i) & 1));
                        if (!ok) break;
                        tc_fence_after();
                        if (leader) {
                            weighted(m, i, (done[m] + i) & 1, ring + sv * C::SLOT);
                            if (C::P_APART || i + 1 == n) umma_commit(&sh->o_full[m]);
                        }
                        __syncwarp();
                        if (!C::P_APART && i + 1 < n) {
                            ok = __all_sync(0xffffffffu, bar_wait(sh, &sh->k_full[sk], use_parity(gk)));
                            if (ok) ok = issue_scores(m, sk, i + 1);
                        }
                    }
                    if (ok && leader) {
                        umma_commit(&sh->empty[sv]);
                        if (!C::P_APART && more) {
                            umma_commit(&sh->empty[sk]);
                            if (i + 2 == nt) umma_commit(&sh->q_empty);
                        }
                    }
                    __syncwarp();
                }
                g += 2 * nt, done[0] += n0, done[1] += n1;
                leave_item(k);
            }
        } else if (warp == 2) {
            // ── V check ──────────────────────────────────────────────────────────
            constexpr uint32_t EXP = std::is_same<T16, __nv_bfloat16>::value ? 0x7F807F80u : 0x7C007C00u;  // exponent bits, and
            constexpr uint32_t ONE = std::is_same<T16, __nv_bfloat16>::value ? 0x00800080u : 0x04000400u;  // their lowest one
            uint32_t g0 = 0;
            bool ok = true;
            for (uint32_t k = 0; ok; k++) {
                const Item* it = next_item(k);
                if (!it) break;
                Item* notes = &sh->item[k % PR_ITEMS];
                const int nt = it->nt(), first_masked = it->template first_masked<NK>();
                for (int i = 0; i < nt; i++) {
                    const uint32_t g = g0 + 2 * i + 1, s = g % NS;
                    if (!(ok = __all_sync(0xffffffffu, bar_wait(sh, &sh->v_full[s], use_parity(g))))) break;
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
                        if (PLANES == 1 && lane < 4) notes->mask[i - first_masked][lane] = lane == 0 ? found[0] : lane == 1 ? found[1] : lane == 2 ? found[2] : found[3];
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                    __syncwarp();
                    if (lane == 0) bar_arrive(&sh->ready[s]);
                }
                g0 += 2 * nt;
                __syncwarp();
                if (lane == 0 && ok) bar_arrive(&sh->checked[k % PR_ITEMS]);
                leave_item(k);
            }
        }
    } else {
        // ── softmax: one row per thread ──────────────────────────────────────
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int m = (warp - 4) >> 2, r = (warp & 3) * 32 + lane, j = m * a.tile_tokens + r / a.group;
        const uint32_t t_s = tmem + m * 256 + C::S_COL + ((uint32_t)((warp & 3) * 32) << 16), t_p = t_s + C::P_COL, t_o = t_s + C::O_COL;
        const float NEG = __int_as_float(0xFF800000);
        uint32_t done = 0, items = 0;  // tiles and items with keys of this row tile so far
        float next_q = 0.0f;           // f32: the power of two taken out of this row of the item that comes next
        // f32: this thread's row of an item's Q.  It has come as 32 elements to a 128-byte column, whose bytes become the 32 high and the 32 low
        // parts.  Loops stay loops here and below: code that runs once per item is fetched anew each time, and unrolled it took longer
        // to fetch than to run (3000 to 7000 cycles for this).
        uint32_t raw = 0;  // items whose Q this row tile has taken
        auto write_q = [&]() -> float {
            if (!bar_wait(sh, &sh->q_raw[m], raw & 1)) return 0.0f;
            raw++;
            const uint32_t row = q_smem + m * PLANES * C::QBYTES + r * 128;
            float top = 0.0f;  // (an infinity or NaN makes the row's results NaN in any case)
            float v[32];
#pragma unroll 1
            for (int c = 0; c < 2 * C::CH; c++) {
#pragma unroll
                for (int x = 0; x < 8; x++) lds_4(row + c * PR_ROWS * 128 + (x ^ (r & 7)) * 16, v + 4 * x);
#pragma unroll
                for (int x = 0; x < 32; x++) top = fmaxf(top, fabsf(v[x]));
            }
            const float f = to_range(top);
            const f32x2 f2 = pack2(f, f), minus = pack2(-1.0f, -1.0f);
#pragma unroll 1
            for (int c = 0; c < 2 * C::CH; c++) {
#pragma unroll
                for (int x = 0; x < 8; x++) lds_4(row + c * PR_ROWS * 128 + (x ^ (r & 7)) * 16, v + 4 * x);
#pragma unroll
                for (int x = 0; x < 4; x++) {  // eight values, 16 bytes of each part
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        const f32x2 q2 = mul2(pack2(v[8 * x + 2 * y], v[8 * x + 2 * y + 1]), f2);
                        float q0, q1, l0, l1;
                        unpack2(q2, q0, q1);
                        const float h0 = __uint_as_float(__float_as_uint(q0) & 0xFFFFE000u), h1 = __uint_as_float(__float_as_uint(q1) & 0xFFFFE000u);
                        unpack2(fma2(pack2(h0, h1), minus, q2), l0, l1);
                        hi[y] = pack16<T16>(h0, h1), lo[y] = pack16<T16>(l0, l1);
                    }
                    sts_4(row + c * PR_ROWS * 128 + (x ^ (r & 7)) * 16, hi);
                    sts_4(row + c * PR_ROWS * 128 + ((x + 4) ^ (r & 7)) * 16, lo);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) bar_arrive(&sh->q_full[m]);
            return __fdiv_rn(1.0f, f);
        };
        bool ok = true;
        bool written = false;  // f32: the coming item's Q is in its place
        for (uint32_t k = 0;; k++) {
            const Item* it = next_item(k);
            if (!it) break;
            const int head = it->kvh * a.group + r % a.group, n = it->n_tiles[m], nt = it->nt(), first_masked = it->template first_masked<NK>();
            const bool real = r < a.tile_tokens * a.group && j < it->tokens;
            const int limit = real ? it->visible(j) : 0;
            float row_max = NEG, row_sum = 0.0f;
            bool bad = false;  // f32: some tile has values that are not finite
            float o[C::O_IN_TMEM ? 1 : HDP];
            // 16 bits: O of PR_CARRY tiles at a time, added up outside the tensor core, behind it the maximum that the sum goes by (local memory: few
            // calls come here, and it takes no registers from the others)
            float carry[C::O_IN_TMEM ? HDP + 1 : 1];
            carry[0] = 0.0f;
            auto with_carry = [&](int c, float (&x)[32]) {
                if constexpr (C::O_IN_TMEM) {
                    const float was = carry[HDP], f = was == row_max ? 1.0f : exp2_approx(was - row_max);
#pragma unroll
                    for (int d = 0; d < 32; d++) x[d] = fmaf(carry[c + d], f, x[d]);
                }
            };
            if constexpr (C::O_IN_TMEM) {
                for (int first = 0; first < n && ok; first += PR_CARRY) {
                    if (first > 0) {  // (behind the P V of the tile before: with P over S by this tile's S, with P apart by its own sign)
                        if (!(ok = __all_sync(0xffffffffu, C::P_APART ? bar_wait(sh, &sh->o_full[m], (done + first - 1) & 1) : bar_wait(sh, &sh->s_full[m], (done + first) & 1)))) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < HDP; c += 32) {
                            float x[32];
                            tmem_ld32(t_o + c, x);
                            tmem_ld_wait();
                            if (first > PR_CARRY) with_carry(c, x);
#pragma unroll
                            for (int d = 0; d < 32; d++) carry[c + d] = x[d], x[d] = 0.0f;
                            tmem_st32(t_o + c, x);
                        }
                        carry[HDP] = row_max;
                    }
                    for (int i = first; i < min(n, first + PR_CARRY) && ok; i++) {
                        if (!(ok = __all_sync(0xffffffffu, bar_wait(sh, &sh->s_full[m], (done + i) & 1)))) break;
                        tc_fence_after();
                        float s[NK];
#pragma unroll
                        for (int c = 0; c < NK / 32; c++) tmem_ld32(t_s + 32 * c, s + 32 * c);
                        tmem_ld_wait();
                        if (C::P_APART) {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) bar_arrive(&sh->s_read[m]);
                        }
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
                        // P V of the tile before is done: with P over S by the order of the tensor core's work, with P apart by this wait
                        if (C::P_APART && i > 0 && !(ok = __all_sync(0xffffffffu, bar_wait(sh, &sh->o_full[m], (done + i - 1) & 1)))) break;
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
                        // f16: 2^7 times the weights, at most 2^15 then: those down to 2^-32 of the maximum stay in its range.  bf16, which has f32's: 2^-8
                        // of them, at most 1, so that values near its end stay in range.
                        constexpr float LIFT = std::is_same<T16, __half>::value ? 7.0f : -PR_LAZY;
                        float scale = a.scale_log2, base = (row_max == NEG ? 0.0f : -row_max) + LIFT;
                        if (__builtin_expect(__any_sync(0xffffffffu, coarse(row_max)), 0)) {  // (rarely: one look for the warp)
                            if (coarse(row_max)) {
#pragma unroll
                                for (int c = 0; c < NK; c++) s[c] = __fsub_rn(__fmul_rn(s[c], scale), row_max);
                                scale = 1.0f, base = LIFT;
                            }
                        }
                        const f32x2 base2 = pack2(base, base), scale2 = pack2(scale, scale);
                        f32x2 sum[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
#pragma unroll
                        for (int c = 0; c < NK / 32; c++) {
                            uint32_t p[16];
#pragma unroll
                            for (int x = 0; x < 16; x++) {
                                float p0, p1;
                                unpack2(fma2(pack2(s[32 * c + 2 * x], s[32 * c + 2 * x + 1]), scale2, base2), p0, p1);
                                p0 = exp2_approx(p0), p1 = exp2_approx(p1);
                                sum[x & 1] = add2(sum[x & 1], pack2(p0, p1));
                                p[x] = pack16<T16>(p0, p1);
                            }
                            tmem_st16(t_p + 16 * c, p);
                        }
                        {
                            float s0, s1;
                            unpack2(add2(sum[0], sum[1]), s0, s1);
                            row_sum += s0 + s1;
                        }
                        tmem_st_wait();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) bar_arrive(&sh->p_ready[m]);
                    }
                }
            } else {
                if (n > 0 && !written) next_q = write_q();
                written = false;
#pragma unroll
                for (int d = 0; d < HDP; d++) o[d] = 0.0f;
                const float row_scale = __fmul_rn(next_q, a.scale_log2);
                const float* k_inv = a.k_inv + (size_t)it->key_slot0 * a.p.n_kv + it->kvh;
                const float* v_inv = a.v_inv + (size_t)it->key_slot0 * a.p.n_kv + it->kvh;
                float rescale = 0.0f;  // of what `o` holds, for the tile whose P V is still in tensor memory
                float k_next = n > 0 ? k_inv[0] : 0.0f, v_now = 0.0f, v_next = n > 0 ? v_inv[0] : 0.0f;  // (a tile ahead)
                auto take_o = [&](int i, float f) {
                    const f32x2 f2 = pack2(f, f), rescale2 = pack2(rescale, rescale);
#pragma unroll
                    for (int c = 0; c < HDP; c += 32) {
                        float x[32];
                        tmem_ld32(t_o + (C::O_BUFS == 2 ? ((done + i) & 1) * HDP : 0) + c, x);
                        tmem_ld_wait();
#pragma unroll
                        for (int d = 0; d < 32; d += 2)
                            unpack2(fma2(pack2(x[d], x[d + 1]), f2, mul2(pack2(o[c + d], o[c + d + 1]), rescale2)), o[c + d], o[c + d + 1]);
                    }
                };
                for (int i = 0; i < n && ok; i++) {
                    const float k_now = k_next, v_before = __fmul_rn(fabsf(v_now), PR_DOWN);
                    const bool k_far = k_now < 0.0f, v_far = v_next < 0.0f;
                    float scale = k_far ? a.scale_log2 : __fmul_rn(row_scale, k_now);
                    v_now = v_next;
                    if (i + 1 < n) k_next = k_inv[(size_t)(i + 1) * a.p.n_kv], v_next = v_inv[(size_t)(i + 1) * a.p.n_kv];
                    if (!(ok = __all_sync(0xffffffffu, bar_wait(sh, &sh->s_full[m], (done + i) & 1)))) break;
                    tc_fence_after();
                    const int seen = limit - i * NK;
                    const bool masked = __any_sync(0xffffffffu, seen < NK);
                    if (__builtin_expect(k_far, 0)) {  // S without its powers of two (products with which are exact), far keys' anew
#pragma unroll 1
                        for (int c = 0; c < NK / 32; c++) {
                            float s[32];
                            tmem_ld32(t_s + 32 * c, s);
                            tmem_ld_wait();
#pragma unroll
                            for (int x = 0; x < 32; x++) s[x] = __fmul_rn(__fmul_rn(s[x], next_q), -k_now);
                            tmem_st32(t_s + 32 * c, s);
                        }
                        tmem_st_wait();
                        const Item* at = aside(it);
                        const int row = aside(r), width = aside(hd);
                        const uint32_t* far = a.k_far + far_tile(a, at, i);
                        const float* q = reinterpret_cast<const float*>(a.p.q) + (size_t)(at->token0 + m * a.tile_tokens + row / a.group) * a.p.q_stride +
                                         (size_t)(at->kvh * a.group + row % a.group) * width;
                        const float* k0 = reinterpret_cast<const float*>(a.p.k) + (size_t)(at->key0 + i * NK) * a.p.k_stride + (size_t)at->kvh * width;
#pragma unroll 1
                        for (int w = 0; w < NK / 32; w++)
#pragma unroll 1
                            for (uint32_t bits = far[w]; bits; bits &= bits - 1) {
                                const int t = 32 * w + __ffs(bits) - 1;
                                float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
                                if (t < seen) {
                                    const float* key = k0 + (size_t)t * a.p.k_stride;
#pragma unroll 2
                                    for (int d = 0; d < width; d += 4) {
                                        const float4 x = *reinterpret_cast<const float4*>(q + d), y = *reinterpret_cast<const float4*>(key + d);
                                        sum.x = fmaf(x.x, y.x, sum.x), sum.y = fmaf(x.y, y.y, sum.y), sum.z = fmaf(x.z, y.z, sum.z), sum.w = fmaf(x.w, y.w, sum.w);
                                    }
                                }
                                __syncwarp();
                                tmem_st1(t_s + t, (sum.x + sum.y) + (sum.z + sum.w));
                            }
                        tmem_st_wait();
                    }
                    float tops[4] = {NEG, NEG, NEG, NEG};
#pragma unroll 1
                    for (int c = 0; c < NK / 32; c++) {
                        float s[32];
                        tmem_ld32(t_s + 32 * c, s);
                        tmem_ld_wait();
                        if (masked) {
#pragma unroll
                            for (int x = 0; x < 32; x++)
                                if (x >= seen - 32 * c) s[x] = NEG;
                        }
#pragma unroll
                        for (int x = 0; x < 32; x++) tops[x & 3] = fmaxf(tops[x & 3], s[x]);
                    }
                    const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                    if (C::O_BUFS == 1 && i > 0) take_o(i - 1, v_before);
                    const float new_max = fmaxf(row_max, __fmul_rn(top, scale));
                    const float f = row_max == NEG ? 0.0f : exp2_approx(row_max - new_max);
                    // weights up to 2^8 in the products, so that the low parts of small ones stay in f16's range; in the sums up to 1 again, so that
                    // values near the end of f32 stay in its range
                    float base = new_max == NEG ? 0.0f : PR_LAZY - new_max;
                    row_max = new_max;
                    if (__builtin_expect(__any_sync(0xffffffffu, coarse(row_max)), 0)) {
                        const bool mine = coarse(row_max);
#pragma unroll 1
                        for (int c = 0; c < NK / 32; c++) {
                            float s[32];
                            tmem_ld32(t_s + 32 * c, s);
                            tmem_ld_wait();
#pragma unroll
                            for (int x = 0; x < 32; x++) s[x] = mine ? __fsub_rn(__fmul_rn(s[x], scale), row_max) : s[x];
                            tmem_st32(t_s + 32 * c, s);
                        }
                        tmem_st_wait();
                        if (mine) scale = 1.0f, base = PR_LAZY;
                    }
                    if (__builtin_expect(v_far, 0)) {  // the far keys' weighted values; the tensor core's product has zeros there
                        if (C::O_BUFS == 2 && i > 0) take_o(i - 1, v_before);
#pragma unroll
                        for (int d = 0; d < HDP; d++) o[d] = __fmul_rn(o[d], f);
                        const Item* at = aside(it);
                        const int width = aside(hd);
                        const uint32_t *far = a.v_far + far_tile(a, at, i), *not_finite = a.v_bad + far_tile(a, at, i);
                        const float* v0 = reinterpret_cast<const float*>(a.p.v) + (size_t)(at->key0 + i * NK) * a.p.v_stride + (size_t)at->kvh * width;
#pragma unroll 1
                        for (int w = 0; w < NK / 32; w++)
#pragma unroll 1
                            for (uint32_t bits = (bad |= not_finite[w] != 0, far[w]); bits; bits &= bits - 1) {
                                const int t = 32 * w + __ffs(bits) - 1;
                                const float score = tmem_ld1(t_s + t);
                                tmem_ld_wait();
                                if (t < seen) {
                                    const float weight = __fmul_rn(exp2_approx(fmaf(score, scale, base)), PR_DOWN);
                                    const float* value = v0 + (size_t)t * a.p.v_stride;
#pragma unroll
                                    for (int d = 0; d < HDP; d += 4)
                                        if (d < width) {
                                            const float4 y = finite(*reinterpret_cast<const float4*>(value + d));
                                            o[d] = fmaf(weight, y.x, o[d]), o[d + 1] = fmaf(weight, y.y, o[d + 1]);
                                            o[d + 2] = fmaf(weight, y.z, o[d + 2]), o[d + 3] = fmaf(weight, y.w, o[d + 3]);
                                        }
                                }
                                __syncwarp();
                            }
                    }
                    const f32x2 base2 = pack2(base, base), scale2 = pack2(scale, scale), minus = pack2(-1.0f, -1.0f);
                    f32x2 sum[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
#pragma unroll 1
                    for (int c = 0; c < NK / 32; c++) {
                        float s[32];
                        tmem_ld32(t_s + 32 * c, s);
                        tmem_ld_wait();
                        uint32_t hi[16], lo[16];
#pragma unroll
                        for (int x = 0; x < 16; x++) {
                            float p0, p1, l0, l1;
                            unpack2(fma2(pack2(s[2 * x], s[2 * x + 1]), scale2, base2), p0, p1);
                            if (masked) {
                                if (2 * x >= seen - 32 * c) p0 = NEG;
                                if (2 * x + 1 >= seen - 32 * c) p1 = NEG;
                            }
                            const f32x2 p2 = pack2(p0 = exp2_approx(p0), p1 = exp2_approx(p1));
                            sum[x & 1] = add2(sum[x & 1], p2);
                            const float h0 = __uint_as_float(__float_as_uint(p0) & 0xFFFFE000u);  // 11 bits: exact in f16
                            const float h1 = __uint_as_float(__float_as_uint(p1) & 0xFFFFE000u);
                            unpack2(fma2(pack2(h0, h1), minus, p2), l0, l1);
                            hi[x] = pack16<T16>(h0, h1);
                            lo[x] = pack16<T16>(l0, l1);
                        }
                        tmem_st16(t_p + 32 * c, hi);
                        tmem_st16(t_p + 32 * c + 16, lo);
                    }
                    {
                        float s0, s1;
                        unpack2(add2(sum[0], sum[1]), s0, s1);
                        row_sum = fmaf(row_sum, f, __fmul_rn(s0 + s1, PR_DOWN));
                    }
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(&sh->p_ready[m]);
                    if (C::O_BUFS == 2 && i > 0 && !v_far) take_o(i - 1, v_before);
                    rescale = v_far ? 1.0f : f;
                }
                if (n > 0 && ok) {
                    // the next item's Q while the last P V runs (all of this one's scores have been computed)
                    const Item* then = next_item(k + 1);
                    if (then && then->n_tiles[m] > 0) {
                        next_q = write_q();
                        written = true;
                    }
                    if ((ok = __all_sync(0xffffffffu, bar_wait(sh, &sh->o_full[m], items & 1)))) {
                        tc_fence_after();
                        take_o(n - 1, __fmul_rn(fabsf(v_now), PR_DOWN));
                    }
                }
            }
            if (C::O_IN_TMEM && n > 0 && ok) {
                ok = __all_sync(0xffffffffu, bar_wait(sh, &sh->o_full[m], (C::P_APART ? done + n - 1 : items) & 1));
                tc_fence_after();
            }
            ok = ok && __all_sync(0xffffffffu, bar_wait(sh, &sh->checked[k % PR_ITEMS], (k / PR_ITEMS) & 1));

            // ── the rows: quotient, rounding, values that are not finite ─────
            const float inv = limit > 0 && row_sum != 0.0f ? __fdiv_rn(1.0f, row_sum) : 0.0f;  // (no weight at all: zeros, as without a key)
            const size_t out_row = (size_t)(it->token0 + j) * a.p.n_heads + head, part_row = (size_t)it->part * a.p.n_tokens * a.p.n_heads + out_row;
            T* out = reinterpret_cast<T*>(a.p.out) + out_row * hd;
            float* sums = a.part_o + part_row * hd;
            const bool split = a.splits > 1;
            if (split && real && ok) *reinterpret_cast<float2*>(a.part_ml + part_row * 2) = make_float2(limit > 0 && n > 0 ? row_max : NEG, limit > 0 && n > 0 ? row_sum : 0.0f);
            auto write_32 = [&](int c, float (&x)[32]) {
                if (split) {
#pragma unroll
                    for (int d = 0; d < 32; d += 8)  // (head_dim is a multiple of 8: rows start on 32-byte boundaries)
                        if (c + d < hd) {
#pragma unroll
                            for (int u = 0; u < 8; u++) x[d + u] = limit > 0 && n > 0 ? x[d + u] : 0.0f;
                            asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(sums + c + d), "f"(x[d]), "f"(x[d + 1]), "f"(x[d + 2]),
                                         "f"(x[d + 3]), "f"(x[d + 4]), "f"(x[d + 5]), "f"(x[d + 6]), "f"(x[d + 7])
                                         : "memory");
                        }
                    return;
                }
#pragma unroll
                for (int d = 0; d < 32; d++) x[d] = limit > 0 ? __fmul_rn(x[d], inv) : 0.0f;
                constexpr int V = 16 / (int)sizeof(T);
#pragma unroll
                for (int d = 0; d < 32; d += 2 * V) {
                    uint32_t w[8];
#pragma unroll
                    for (int u = 0; u < 8; u++)
                        if constexpr (sizeof(T) == 4)
                            w[u] = __float_as_uint(x[d + u]);
                        else
                            w[u] = pack16<T>(x[d + 2 * u], x[d + 2 * u + 1]);
                    T* to = out + c + d;
                    // A row is a thread's: 32 bytes at a time are whole sectors
                    if (a.wide_rows && c + d + 2 * V <= hd)
                        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                                     "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                                     : "memory");
                    else {
                        if (c + d < hd) *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
                        if (c + d + V < hd) *reinterpret_cast<uint4*>(to + V) = make_uint4(w[4], w[5], w[6], w[7]);
                    }
                }
            };
            if constexpr (C::O_IN_TMEM) {
#pragma unroll 1
                for (int c = 0; c < HDP; c += 32) {
                    float x[32];
                    if (n > 0) {  // (uniform in the warp)
                        tmem_ld32(t_o + c, x);
                        tmem_ld_wait();
                        if (n > PR_CARRY) with_carry(c, x);
                    }
                    if (real && ok) write_32(c, x);
                }
            } else if (real && ok) {
#pragma unroll
                for (int c = 0; c < HDP; c += 32) {
                    float x[32];
#pragma unroll
                    for (int d = 0; d < 32; d++) x[d] = o[C::O_IN_TMEM ? 0 : c + d];
                    write_32(c, x);
                }
            }
            auto add_not_finite = [&](int first, uint32_t bits) {  // of the keys from `first` on that have a bit
                for (; bits; bits &= bits - 1) {
                    const int t = first + __ffs(bits) - 1;
                    if (t >= limit || !ok) continue;
                    const T* v = reinterpret_cast<const T*>(a.p.v) + (size_t)(it->key0 + t) * a.p.v_stride + (size_t)it->kvh * hd;
#pragma unroll 1
                    for (int d = 0; d < hd; d++) {
                        const float y = to_f32(v[d]);
                        if (fabsf(y) <= MAX_F32) continue;
                        if (split)
                            sums[d] = __fadd_rn(sums[d], y);
                        else
                            out[d] = from_f32<T>(__fadd_rn(to_f32(out[d]), y));
                    }
                }
            };
            if constexpr (PLANES == 1) {
                for (int i = first_masked; i < nt; i++)
#pragma unroll 1
                    for (int w = 0; w < NK / 32; w++) add_not_finite(i * NK + w * 32, it->mask[i - first_masked][w]);
            } else if (bad) {
#pragma unroll 1
                for (int i = 0; i < n; i++) {
                    const size_t tile = far_tile(a, it, i);
                    if (a.v_inv[tile / FAR_WORDS] >= 0.0f) continue;
#pragma unroll 1
                    for (int w = 0; w < NK / 32; w++) add_not_finite(i * NK + w * 32, a.v_bad[tile + w]);
                }
            }
            tc_fence_before();  // (tensor memory has been read before the next P V, which waits for p_ready)
            done += n, items += n > 0 ? 1 : 0;
            leave_item(k);
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        if (sh->abort) {
            settle();
            Deal<NK> deal(a);
            Item it;
            while (deal.next(a, it)) {  // no row is left without a sign of it
                for (int i = lane; i < it.tokens * a.group * hd; i += 32) {
                    const size_t row = (size_t)(it.token0 + i / (a.group * hd)) * a.p.n_heads + it.kvh * a.group + i % (a.group * hd) / hd;
                    if (a.splits > 1)
                        a.part_ml[((size_t)it.part * a.p.n_tokens * a.p.n_heads + row) * 2 + 1] = __int_as_float(0x7FC00000);
                    else
                        reinterpret_cast<T*>(a.p.out)[row * hd + i % hd] = from_f32<T>(__int_as_float(0x7FC00000));
                }
            }
        }
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

struct SplitArgs {
    Prompts p;
    __half* to[2];  // keys, values: [2][rows][heads * head_dim]
    float* inv[2];
    uint32_t *far[2], *v_bad;
    int lanes;      // of a row: head_dim / 4 rounded up to a power of two
};
constexpr int SP_THREADS = 256;

// A tile of K or V per CTA, held in registers between the search for its rows' largest magnitudes and its parts.  Bound: HBM (4 bytes in, 4 out
// per element), the launch for short prompts.
// The tile's power of two is that of its largest row, if no row lies below 2^-14 of it (its largest element then has 24 bits or more above the
// parts' 2^-25); elements that are not finite do not count.  Otherwise it is the row's from which most rows lie within 2^-14, the larger of equals; the others are far.
template <int NK>
__global__ void __launch_bounds__(SP_THREADS) k_split(const __grid_constant__ SplitArgs a) {
    pdl_trigger();
    pdl_wait();
    __shared__ uint2 red[SP_THREADS / 32];
    __shared__ uint32_t row_top[NK], row_bad[NK];  // bits of the rows' largest finite magnitudes; whether they have others
    __shared__ unsigned long long best[SP_THREADS / 32];
    const int hd = a.p.head_dim, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int val = blockIdx.x & 1, kvh = (blockIdx.x >> 1) % a.p.n_kv, slot = (blockIdx.x >> 1) / a.p.n_kv;
    const int32_t* ks = a.p.key_starts ? a.p.key_starts : a.p.starts;
    const int seq = find_seq(ks, a.p.n_seqs, a.p.n_keys, NK, slot);
    if (seq < 0) return;
    const int k0 = max(0, min(ks[seq], a.p.n_keys)), k1 = max(k0, min(ks[seq + 1], a.p.n_keys));
    const int first = k0 + (slot - (k0 / NK + seq)) * NK, rows = min(NK, k1 - first);
    if (rows <= 0) return;
    const size_t stride = val ? a.p.v_stride : a.p.k_stride, dim = (size_t)a.p.n_kv * hd, plane = (size_t)a.p.n_keys * dim;
    const int piece = threadIdx.x & (a.lanes - 1), row0 = threadIdx.x / a.lanes, step = SP_THREADS / a.lanes;
    const float* src = (const float*)(val ? a.p.v : a.p.k) + (size_t)first * stride + (size_t)kvh * hd + 4 * piece;
    const bool in = 4 * piece < hd;
    constexpr int MOST = NK * (NK == 128 ? 16 : 32) / SP_THREADS;  // rows of a thread, at most (heads of up to 64 have tiles of 128 keys)
    float4 x[MOST];
#pragma unroll
    for (int i = 0; i < MOST; i++) {
        const int row = row0 + i * step;
        x[i] = in && row < rows ? *reinterpret_cast<const float4*>(src + row * stride) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    // Bits of magnitudes: their difference counts powers of two.  First by the threads' pieces of rows, zeros left out: where none of them lies below
    // the window, no row does.
    constexpr uint32_t WINDOW = 14u << 23, INF = 0x7F800000u;
    uint32_t most = 0, least = 0xFFFFFFFFu;
#pragma unroll
    for (int i = 0; i < MOST; i++) {
        const uint32_t top = magnitude(x[i]);
        most = max(most, top), least = min(least, top - 1);
    }
    most = __reduce_max_sync(0xffffffffu, most), least = __reduce_min_sync(0xffffffffu, least);
    if (lane == 0) red[warp] = make_uint2(most, least);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SP_THREADS / 32; w++) most = max(most, red[w].x), least = min(least, red[w].y);
    const bool bad_rows = most >= INF;  // rows with elements that are not finite
    bool far_rows = bad_rows || (most != 0 && most - (least + 1) > WINDOW);
    if (far_rows) {  // by whole rows, their finite elements
#pragma unroll
        for (int i = 0; i < MOST; i++) {
            uint32_t bad = magnitude(x[i]) >= INF;
            x[i] = finite(x[i]);
            uint32_t top = magnitude(x[i]);
            for (int o = a.lanes / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o)), bad |= __shfl_xor_sync(0xffffffffu, bad, o);
            if (piece == 0 && row0 + i * step < NK) row_top[row0 + i * step] = top, row_bad[row0 + i * step] = bad;
        }
        __syncthreads();
        most = 0, least = 0xFFFFFFFFu;
        for (int r = lane; r < NK; r += 32) most = max(most, row_top[r]), least = min(least, row_top[r] - 1);
        most = __reduce_max_sync(0xffffffffu, most), least = __reduce_min_sync(0xffffffffu, least);
        far_rows = most != 0 && most - (least + 1) > WINDOW;
    }
    if (far_rows) {
        unsigned long long mine = 0;
        if (threadIdx.x < NK) {
            const uint32_t top = row_top[threadIdx.x];
            uint32_t count = 0;
            for (int r = 0; r < NK; r++) count += row_top[r] != 0 && top - row_top[r] <= WINDOW;
            mine = top ? (unsigned long long)count << 32 | top : 0;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
        if (lane == 0) best[warp] = mine;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < SP_THREADS / 32; w++) mine = max(mine, best[w]);
        most = (uint32_t)mine;
    }
    const float f = to_range(__uint_as_float(most));
    auto far_row = [&](int row) {  // (above the window: the difference wraps)
        return (far_rows && row_top[row] != 0 && most - row_top[row] > WINDOW) || (bad_rows && !val && row_bad[row]);
    };
    const size_t tile = (size_t)slot * a.p.n_kv + kvh;
    const bool marked = far_rows || bad_rows;
    if (marked && threadIdx.x < NK) {
        const uint32_t far = __ballot_sync(0xffffffffu, far_row(threadIdx.x)), bad = __ballot_sync(0xffffffffu, bad_rows && row_bad[threadIdx.x]);
        if (lane == 0) {
            a.far[val][tile * FAR_WORDS + warp] = far;
            if (val) a.v_bad[tile * FAR_WORDS + warp] = bad;
        }
    }
    __half* dst = a.to[val] + (size_t)first * dim + (size_t)kvh * hd + 4 * piece;
#pragma unroll
    for (int i = 0; i < MOST; i++) {
        const int row = row0 + i * step;
        if (in && row < rows) {
            uint2 hi, lo;
            if (marked && far_row(row)) x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            split4(x[i], f, hi, lo);
            *reinterpret_cast<uint2*>(dst + row * dim) = hi;
            *reinterpret_cast<uint2*>(dst + row * dim + plane) = lo;
        }
    }
    if (threadIdx.x == 0) a.inv[val][tile] = marked ? -__fdiv_rn(1.0f, f) : __fdiv_rn(1.0f, f);
}

// The parts of the rows' keys, added up in their order: four values of a row per thread (threadIdx.x), all parts' loads under way together.
constexpr int JOIN_THREADS = 256, MAX_SPLITS = 8;
template <class T>
__global__ void __launch_bounds__(JOIN_THREADS) k_join(const __grid_constant__ PromptArgs a) {
    pdl_trigger();
    pdl_wait();
    const int hd = a.p.head_dim, d = threadIdx.x * 4;
    const size_t rows = (size_t)a.p.n_tokens * a.p.n_heads, first = (size_t)max(0, min(a.p.starts[0], a.p.n_tokens)) * a.p.n_heads;
    const size_t last = (size_t)max(0, min(a.p.starts[a.p.n_seqs], a.p.n_tokens)) * a.p.n_heads;
    const size_t row = (size_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (row < first || row >= last) return;  // (a row of no sequence)
    float2 ml[MAX_SPLITS];
    float4 x[MAX_SPLITS];
    float m = __int_as_float(0xFF800000);
#pragma unroll
    for (int s = 0; s < MAX_SPLITS; s++) {
        ml[s] = make_float2(m, 0.0f), x[s] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (s < a.splits) {
            ml[s] = *reinterpret_cast<const float2*>(a.part_ml + (s * rows + row) * 2);
            x[s] = *reinterpret_cast<const float4*>(a.part_o + (s * rows + row) * hd + d);
        }
    }
#pragma unroll
    for (int s = 0; s < MAX_SPLITS; s++) m = fmaxf(m, ml[s].x);
    float l = 0.0f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int s = 0; s < MAX_SPLITS; s++)
        if (s < a.splits) {
            const float f = ml[s].x == m ? 1.0f : exp2_approx(ml[s].x - m);
            l = fmaf(ml[s].y, f, l);
            auto add = [f](float y, float to) { return fmaf(y, fabsf(y) <= MAX_F32 ? f : 1.0f, to); };  // (an infinite value has no factor)
            o = make_float4(add(x[s].x, o.x), add(x[s].y, o.y), add(x[s].z, o.z), add(x[s].w, o.w));
        }
    const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
    T* out = reinterpret_cast<T*>(a.p.out) + row * hd + d;
    if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4*>(out) = make_float4(__fmul_rn(o.x, inv), __fmul_rn(o.y, inv), __fmul_rn(o.z, inv), __fmul_rn(o.w, inv));
    else
        *reinterpret_cast<uint2*>(out) = make_uint2(pack16<T>(__fmul_rn(o.x, inv), __fmul_rn(o.y, inv)), pack16<T>(__fmul_rn(o.z, inv), __fmul_rn(o.w, inv)));
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
// Rows [planes][rows][heads][head_dim]; box: 128 bytes of a head (zeros behind head_dim) x box_heads x box_rows, 128-byte swizzle.
cudaError_t encode_heads(const void* base, int dtype, int hd, int heads, int rows, int planes, size_t stride, int box_heads, int box_rows, CUtensorMap* out) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return cudaErrorNotSupported;
    const cuuint64_t size = (cuuint64_t)dtype_bytes(dtype), dims[4] = {(cuuint64_t)hd, (cuuint64_t)heads, (cuuint64_t)rows, (cuuint64_t)planes};
    const cuuint64_t strides[3] = {(cuuint64_t)hd * size, (cuuint64_t)stride * size,
                                   (cuuint64_t)stride * size * (planes > 1 ? (cuuint64_t)rows : 1)};  // (of one plane: any)
    const cuuint32_t box[4] = {(cuuint32_t)(128 / size), (cuuint32_t)box_heads, (cuuint32_t)box_rows, 1}, step[4] = {1, 1, 1, 1};
    const CUtensorMapDataType type = dtype == DT_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : dtype == DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const CUresult r = fn(out, type, 4, const_cast<void*>(base), dims, strides, box,
                          step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

constexpr size_t up128(size_t n) { return (n + 127) & ~(size_t)127; }
int keys_per_tile(const Prompts& p) { return p.dtype == DT_F32 && p.head_dim > 64 ? Cfg<2, 128>::NK : Cfg<1, 64>::NK; }
int places(int rows, int seqs, int block) { return rows / block + seqs + 1; }
int block_tokens(const Prompts& p) { return 2 * (PR_ROWS / (p.n_heads / p.n_kv)); }
// Parts of a block's keys.  An item takes its tiles and about 2.5 more (its first scores, its rows); the launch takes as many items of mean length as
// come to the fullest SM, or the longest one; a join takes three.  The number for which that is least, taking sequences for alike (the sizes decide
// alone, so that the workspace can be asked for).  Of 34 shapes, 1 to 16 sequences of 8 to 4000 tokens behind 0 to 30000 keys, heads of 32 to 128, each timed with
// 1, 2, 3, 4, 5, 6 and 8 parts, it takes 2 % more than the best on average, undivided calls 36 %.  (Four chunks of up to 512 tokens behind 3500 keys: 1,
// 2, 3, 4 parts 129, 115, 112, 114 us.)
int key_splits(const Prompts& p) {
    const int sms = 148, block = block_tokens(p);
    if (p.n_seqs == 0 || p.n_tokens == 0) return 1;
    const double tokens = (double)p.n_tokens / p.n_seqs, keys = (double)p.n_keys / p.n_seqs;
    const double blocks = p.n_seqs == 1 ? std::ceil(tokens / block) : std::max(tokens / block + 0.5, 1.0);  // (the last one half full)
    const double items = blocks * p.n_seqs * p.n_kv;
    const double longest = keys / keys_per_tile(p), mean = std::max(0.0, keys - tokens / 2) / keys_per_tile(p);
    int best = 1;
    double least = 0.0;
    for (int s = 1; s <= MAX_SPLITS && (s == 1 || longest / s >= 2.0); s++) {
        const double cost = std::max(longest / s + 2.5, std::ceil(items * s / sms) * (mean / s + 2.5)) + (s > 1 ? 3.0 : 0.0);
        if (s == 1 || cost < 0.97 * least) least = cost, best = s;
    }
    return best;
}

struct Workspace {
    size_t k = 0, v = 0, k_inv = 0, v_inv = 0, k_far = 0, v_far = 0, v_bad = 0, part_o = 0, part_ml = 0, bytes;
    explicit Workspace(const Prompts& p) {
        const size_t key_slots = (size_t)places(p.n_keys, p.n_seqs, keys_per_tile(p));
        size_t at = 0;
        auto take = [&at](size_t n) {
            const size_t here = at;
            at += up128(n);
            return here;
        };
        if (p.dtype == DT_F32) {
            k = take((size_t)p.n_keys * p.n_kv * p.head_dim * 4);
            v = take((size_t)p.n_keys * p.n_kv * p.head_dim * 4);
            k_inv = take(key_slots * p.n_kv * 4);
            v_inv = take(key_slots * p.n_kv * 4);
            k_far = take(key_slots * p.n_kv * FAR_WORDS * 4);
            v_far = take(key_slots * p.n_kv * FAR_WORDS * 4);
            v_bad = take(key_slots * p.n_kv * FAR_WORDS * 4);
        }
        const int splits = key_splits(p);
        if (splits > 1) {
            part_o = take((size_t)splits * p.n_tokens * p.n_heads * p.head_dim * 4);
            part_ml = take((size_t)splits * p.n_tokens * p.n_heads * 8);
        }
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
    a.waits = serving_waits();
    a.wide_rows = (((uintptr_t)p.out | (size_t)p.head_dim * sizeof(T)) & 31) == 0;
    a.scale_log2 = 1.4426950408889634f / sqrtf((float)p.head_dim);
    const int parts = PLANES == 2 ? DT_F16 : p.dtype;  // what K and V are in
    const void *k = p.k, *v = p.v;
    size_t ks = p.k_stride, vs = p.v_stride;
    const Workspace w(p);
    uint8_t* base = static_cast<uint8_t*>(workspace);
    a.splits = key_splits(p);
    a.part_o = (float*)(base + w.part_o), a.part_ml = (float*)(base + w.part_ml);
    if (PLANES == 2 && p.n_keys > 0) {
        SplitArgs s{p, {(__half*)(base + w.k), (__half*)(base + w.v)}, {(float*)(base + w.k_inv), (float*)(base + w.v_inv)},
                    {(uint32_t*)(base + w.k_far), (uint32_t*)(base + w.v_far)}, (uint32_t*)(base + w.v_bad), 1};
        while (s.lanes * 4 < p.head_dim) s.lanes *= 2;
        const long long ctas = (long long)places(p.n_keys, p.n_seqs, C::NK) * p.n_kv * 2;
        if (ctas > 0x7FFFFFFFll) return cudaErrorInvalidValue;
        g_kernel_launches++;
        if ((e = launch_pdl(st, k_split<C::NK>, dim3((unsigned)ctas), dim3(SP_THREADS), 0, s)) != cudaSuccess) return e;
        k = s.to[0], v = s.to[1];
        ks = vs = (size_t)p.n_kv * p.head_dim;
        a.k_inv = s.inv[0], a.v_inv = s.inv[1];
        a.k_far = s.far[0], a.v_far = s.far[1], a.v_bad = s.v_bad;
    }
    CUtensorMap mq, mk, mv;  // (without any keys none is read)
    if ((e = encode_heads(p.q, p.dtype, p.head_dim, p.n_heads, p.n_tokens, 1, p.q_stride, a.group, a.tile_tokens, &mq)) != cudaSuccess) return e;
    mk = mv = mq;
    if (p.n_keys > 0) {
        if ((e = encode_heads(k, parts, p.head_dim, p.n_kv, p.n_keys, PLANES, ks, 1, C::NK, &mk)) != cudaSuccess) return e;
        if ((e = encode_heads(v, parts, p.head_dim, p.n_kv, p.n_keys, PLANES, vs, 1, C::NK, &mv)) != cudaSuccess) return e;
    }
    int dev = 0, sms = 0;
    if ((e = cudaGetDevice(&dev)) != cudaSuccess) return e;
    if ((e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return e;
    const long long items = (long long)a.slots * p.n_kv * a.splits;
    if (items > 0x7FFFFFFFll - sms) return cudaErrorInvalidValue;
    g_kernel_launches++;
    e = launch_pdl(st, k_attention_prompts<T, PLANES, HDP>, dim3((unsigned)std::min<long long>(items, sms)), dim3(PR_THREADS), C::SMEM, mq, mk, mv, a);
    if (e != cudaSuccess || a.splits == 1) return e;
    g_kernel_launches++;
    const unsigned pieces = (unsigned)p.head_dim / 4, per = JOIN_THREADS / pieces;
    const size_t rows = (size_t)p.n_tokens * p.n_heads;
    return launch_pdl(st, k_join<T>, dim3((unsigned)((rows + per - 1) / per)), dim3(pieces, per), 0, a);
}

}  // namespace

ServingWaits& serving_waits() {
    static thread_local ServingWaits waits;
    return waits;
}

size_t attention_prompts_workspace(const Prompts& p) { return Workspace(p).bytes; }

cudaError_t launch_attention_prompts(cudaStream_t st, const Prompts& p, void* workspace) {
    const bool wide = p.head_dim > 64;
    if (p.dtype == DT_F32) return wide ? launch_typed<float, 2, 128>(st, p, workspace) : launch_typed<float, 2, 64>(st, p, workspace);
    if (p.dtype == DT_F16) return wide ? launch_typed<__half, 1, 128>(st, p, workspace) : launch_typed<__half, 1, 64>(st, p, workspace);
    return wide ? launch_typed<__nv_bfloat16, 1, 128>(st, p, workspace) : launch_typed<__nv_bfloat16, 1, 64>(st, p, workspace);
}

}  // namespace wick

// Attention of many query rows per sequence over the paged 8-bit cache (prompts and chunks of them).
//
// A CTA works on two tiles of 128 query rows of one head of the cache (tokens x the heads that share
// it) and walks the keys in blocks of 128.  Per block and tile:
//     S = Q K^T          tcgen05, both operands fp16 in shared memory, S fp32 in tensor memory
//     P = 2^(S f - M) w  one thread per row: S from tensor memory, P back into its place as fp16
//     O += P V           tcgen05, P from tensor memory, V fp16 in shared memory, O in tensor memory
// The bound is the tensor pipe (4 * 128 * 128 * head_dim operations a block and tile), with the
// exponentials (16 a clock and SM) close behind; bytes from memory hardly count, since a block serves
// 256 rows.  The two tiles keep the pipe busy in turn: one is multiplied while the other is
// exponentiated.  Heads above 128 have one tile, as O of one is half of the tensor memory and the fp16
// tiles of a block are 64 KB each; the warps of the second tile then have nothing to do.
//
// * The tensor cores have no product of fp16 with 8-bit operands, so four warps turn each 8-bit tile,
//   as TMA brought it, into an fp16 tile in the swizzled layout of an operand: exactly, in whatever
//   order of four neighbouring dimensions costs least (Q is laid out to match, O is put right when it
//   is stored).  The same tile layout - 64 dimensions x 128 keys - is K-major for the first product
//   and MN-major for the second, so V needs no transposition.
// * Numerics are those of the rows kernel: queries times a power of two per row, fp32 scores, softmax
//   and sums, weights with their pages' value scales rounded to fp16 in units of a power of two near the
//   row's largest; the running maximum may lag by 2^8, so that O in tensor memory is rescaled only now
//   and then.  Weights are rounded once: outputs in fp16 are off by 0.0003 where rounding the exact result
//   gives 0.0002.  A second part of each weight, as the rows kernel has, brings 0.0002 and costs a second
//   product on the chain: a prompt of 4096 tokens 266 us for 235, the chunk 390 for 333.
// * Work is cut as there: one axis of key blocks over all items, equal shares, pieces joined by a
//   second kernel.
//
// Measured (graph replay): a chunk of 509 tokens behind 32768, 32 over 8 heads of 128, 335 us = 823 TFLOP/s; a
// prompt of 4096 tokens of 32 heads 236 us; 8 prompts of 512 of 12 heads of 64 39 us.  In steady state a block
// of both tiles takes 4850 cycles (counted when the chunk took 328 us), 2048 of them on the tensor pipe: what
// bounds it is the chain of one tile, scores -> 430 cycles for the largest -> 2250 for the weights -> second
// product -> next scores.
// Heads of 256, where nothing overlaps that chain: a prompt of 2048 tokens of 16 heads 128 us (653 in the rows
// kernel), 509 tokens behind 8192, 16 over 4 heads, 165 us = 426 TFLOP/s (570 in the rows kernel).
//
// Warps 0-3 and 4-7: softmax of a tile, a thread a row (the same warps fetch the queries and store the
// outputs); 8-11: conversion; 12: issues the products; 13: copies; 14: scales of the pages; 15: the list of
// what there is to do.
#include "rns_kv.cuh"
#include "rns_ptx.cuh"

namespace rns {

constexpr int kPromptThreads = 512;
constexpr int kConvertWarp = 8, kProductWarp = 12, kCopyWarp = 13, kScaleWarp = 14, kPartWarp = 15;
constexpr int kBlock = 128;               // keys of a block
constexpr int kTileRows = 128;
constexpr float kNoScore = -1.7e38f;      // below every score: "nothing seen yet"
constexpr float kScoreLag = 8.0f;
constexpr int kScaleSlots = 4, kPartSlots = 4;
// What starting and ending an item costs, in blocks: each item takes that much more of the axis that is shared
// out (prompt of 4096 tokens, 32 heads, when it took 229 us: 245 us without, 227 / 229 / 234 with 2 / 3 / 5; 8
// prompts of 512: 42.2 without, 39.0 / 38.4 / 37.1).
constexpr int kItemCost = 3;
// Registers: a softmax thread holds its row's scores of a block.  8 warps of kSoftmaxRegs and 8 of kOtherRegs
// must not exceed what the block was launched with, 16 warps of kLaunchRegs (build.py refuses to build the kernel
// with fewer).
constexpr int kLaunchRegs = 128, kSoftmaxRegs = 176, kOtherRegs = 80;
static_assert(8 * kSoftmaxRegs + 8 * kOtherRegs <= 16 * kLaunchRegs, "register split");

struct PromptParams {
    KvView c;
    KvQuery a;
    int head_tile, token_tile, head_tiles;
    int tiles;                            // of an item: 2, or 1 where O fills the tensor memory
    int min_rows_tokens;                  // sequences with fewer new tokens are left to the rows kernel
    int box_rows;
    float sign;                           // of the softmax scale, which is folded into the queries
    float* partial;                       // [grid][2][256 * (DIM + 2)]
    int32_t* meta;                        // [grid][8]
};

struct PromptItem {
    int b, kv_head, pair;
    int64_t begin;
    int count, length;
    int token0, head0;                    // first token of the pair inside the sequence, first head of its head tile
    int key0, blocks;                     // first key that any row sees, rounded down to a block
    int from[2], to[2];                   // blocks that a tile needs
};

__device__ __forceinline__ bool prompt_sequence(const PromptParams& p, int b, PromptItem& it) {
    const KvSpan s = kv_span(p.c, p.a.lens, p.a.starts, p.a.tokens, b);
    it.b = b; it.begin = s.begin; it.count = s.count; it.length = s.length;
    return s.count >= p.min_rows_tokens && s.count > 0;
}
__device__ __forceinline__ int prompt_pairs(const PromptParams& p, int count) {
    return (count + p.tiles * p.token_tile - 1) / (p.tiles * p.token_tile) * p.head_tiles;
}
__device__ __forceinline__ void prompt_range(const PromptParams& p, PromptItem& it) {
    it.token0 = it.pair / p.head_tiles * p.tiles * p.token_tile;
    it.head0 = it.pair % p.head_tiles * p.head_tile;
    const int base = it.length - it.count;
    int first[2], last[2], low = INT32_MAX, high = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int ta = it.token0 + i * p.token_tile, tb = min(ta + p.token_tile, it.count);
        first[i] = max(0, kv_first_key(p.a, base + ta));
        last[i] = p.a.causal ? base + tb : it.length;
        if (i >= p.tiles || ta >= it.count || base + tb <= 0) last[i] = 0;
        if (last[i] > first[i]) { low = min(low, first[i]); high = max(high, last[i]); }
    }
    it.key0 = high > 0 ? low & ~(kBlock - 1) : 0;
    it.blocks = high > 0 ? (high - it.key0 + kBlock - 1) / kBlock : 1;    // nothing to see: zeros to write
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const bool sees = last[i] > first[i];
        it.from[i] = sees ? (first[i] - it.key0) / kBlock : 0;
        it.to[i] = sees ? (last[i] - it.key0 + kBlock - 1) / kBlock : 0;
    }
}
__device__ __forceinline__ int64_t prompt_head_blocks(const PromptParams& p, PromptItem it) {
    int64_t n = 0;
    const int pairs = prompt_pairs(p, it.count);
    for (it.pair = 0; it.pair < pairs; it.pair += p.head_tiles) {
        prompt_range(p, it);
        n += (int64_t)(it.blocks + kItemCost) * p.head_tiles;
    }
    return n;
}

// What a CTA does is a list of parts: blocks [step, stop) of item after item.  One warp walks the
// axis and publishes the parts; the others read them from shared memory.  On the axis an item is kItemCost
// units of nothing and then its blocks; a part of nothing but those has step == stop.
struct PromptPart {
    PromptItem it;
    int at, used;                         // units of the item's stretch of the axis before this part, and of the part
    int step, stop;
    int live0, live1;                     // blocks of the part that some tile needs (one range: the tiles' meet)
    int mine0[2], mine1[2];               // blocks of it that each tile needs
    int64_t left;                         // units of the CTA from this part on
    int last;                             // no part follows
    int slot;                             // where a piece goes: 0 for the CTA's first blocks, 1 after them

    __device__ __forceinline__ void set(int from, int64_t units) {
        at = from; left = units;
        used = (int)min((int64_t)(it.blocks + kItemCost - at), left);
        step = max(at - kItemCost, 0);
        stop = max(at + used - kItemCost, 0);
        live0 = INT32_MAX; live1 = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            mine0[i] = max(step, it.from[i]);
            mine1[i] = min(stop, it.to[i]);
            if (mine1[i] > mine0[i]) { live0 = min(live0, mine0[i]); live1 = max(live1, mine1[i]); }
            else mine0[i] = mine1[i] = 0;
        }
        if (live1 == 0) live0 = 0;
        last = left <= used;
    }
};
__device__ __forceinline__ void prompt_next(const PromptParams& p, PromptPart& part) {
    PromptItem& it = part.it;
    if (part.stop > part.step) part.slot = 1;
    if (++it.pair >= prompt_pairs(p, it.count)) {
        it.pair = 0;
        if (++it.kv_head >= p.c.kv_heads) {
            it.kv_head = 0;
            int b = it.b + 1;
            while (b < p.c.sequences && !prompt_sequence(p, b, it)) ++b;
        }
    }
    prompt_range(p, it);
    part.set(0, part.left - part.used);
}

template <int DIM> struct PromptShape {
    static constexpr int kParts = DIM / 64;                        // 64-dimension parts of a tile
    static constexpr int kTiles = DIM == 256 ? 1 : 2;              // tiles of an item: S of each and O of each in 512 columns
    static constexpr int kTile = kBlock * DIM * 2;                 // fp16 tile of keys or values
    static constexpr int kRaw = kBlock * DIM;                      // the same in 8 bits
    static constexpr int kRing = DIM == 256 ? 2 : 4, kRawRing = DIM == 64 ? 4 : DIM == 128 ? 2 : 1;
    static constexpr int kQTile = kTileRows * DIM * 2, kQ = kTiles * kQTile;
    static constexpr int kSmem = 1024 + kQ + kRing * kTile + kRawRing * kRaw;
    static constexpr int kPartial = 2 * kTileRows * (DIM + 2);
    static constexpr int kO = 256;                                 // tensor memory: S/P of the tiles at 0 and 128, O from here
};

__device__ __forceinline__ void umma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
          "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
          "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
          "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
          "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld8f(uint32_t taddr, float (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
// Two fp32 operations in one instruction; a pair lives in 64 bits.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float x, float y) { return ((Pair)__float_as_uint(y) << 32) | (Pair)__float_as_uint(x); }
__device__ __forceinline__ float pair_x(Pair p) { return __uint_as_float((uint32_t)p); }
__device__ __forceinline__ float pair_y(Pair p) { return __uint_as_float((uint32_t)(p >> 32)); }
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float prompt_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// fp16, K-major A; B K-major, or MN-major with `b_mn`.  fp32 accumulators.
__device__ __forceinline__ constexpr uint32_t f16_idesc(uint32_t m, uint32_t n, bool b_mn) {
    return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
// MN-major operand with 128-byte swizzle: 64 contiguous MN elements a row, rows along K 128 bytes
// apart, groups of 8 rows `group` bytes apart, blocks of 64 MN elements `block` bytes apart.
__device__ __forceinline__ uint64_t mn_desc(uint32_t addr, uint32_t block, uint32_t group) {
    uint64_t d = 0;
    d |= (uint64_t)((addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(block >> 4) << 16;
    d |= (uint64_t)(group >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
__device__ __forceinline__ uint32_t half_pair_s8(uint32_t x) {
    uint32_t r;                                                   // (x & 0x00ff00ff) ^ 0x64806480 = 1024 + 128 + value
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;\n\tsub.rn.f16x2 %0, %0, %3;" : "=&r"(r) : "r"(x), "r"(0x00ff00ffu), "r"(0x64806480u));
    return r;
}
__device__ __forceinline__ uint32_t half_pair_e4m3(uint32_t x) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(x));
    return r;
}

// Waits of whole warps, bounded by about a second of SM clock.  A poll may be suspended for up to 0.1 ms until
// its phase completes, as most of the 16 warps wait at any time (with the hardware's own limit instead, the chunk
// takes 332 us for 333, a prompt of 4096 tokens 237 for 237).  Waits are kept small: six different programs share
// the instruction cache.
__device__ __forceinline__ bool prompt_poll(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity), "r"(100000u) : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool prompt_wait(uint32_t bar, uint32_t parity, volatile int* abort, int where) {
    bool ok = mbar_try_wait(bar, parity);
    if (!__all_sync(0xffffffffu, ok)) {
        const uint32_t t0 = (uint32_t)clock();
#pragma unroll 1
        while (!ok) {
            ok = prompt_poll(bar, parity);
            if (!ok) {
                if (*abort) break;
                if ((uint32_t)clock() - t0 > 2000000000u) {
                    if (*abort == 0) *abort = where;
                    break;
                }
            }
        }
        ok = __all_sync(0xffffffffu, ok);
    }
    return ok;
}

// What a warp still has on its way lands before it leaves, also when a wait has expired: a wait of its own limit.
__device__ __forceinline__ void prompt_drain(uint32_t bar, uint32_t parity) {
#pragma unroll 1
    for (int i = 0; i < 10000 && !prompt_poll(bar, parity); ++i) {}
}

struct PromptBars {
    uint64_t raw_full[4], raw_empty[4], full[4], empty[4], s_full[2], p_ready[2], o_full[2], q_full[2];
    uint64_t scale_full[kScaleSlots], scale_empty[kScaleSlots], part_full[kPartSlots], part_empty[kPartSlots];
    uint64_t drained;                     // products that were on their way when a wait expired
};
struct PromptScales {
    float key[8], exponent[8], weight[8], back[8];   // of 16 keys each: key scale, and the value scale's kv_value_scale
};

// Bits [lo, hi) of the 32 columns from `at` on: those a row sees.
__device__ __forceinline__ uint32_t prompt_seen(int at, int lo, int hi) {
    const int a = min(max(lo - at, 0), 32), b = min(max(hi - at, 0), 32);
    return (uint32_t)((1ull << b) - 1) & ~(uint32_t)((1ull << a) - 1);
}
// The largest score, with its page's value exponent, of a row of a block of which it sees every column.
__device__ __forceinline__ float prompt_top(uint32_t s_tmem, const PromptScales& sc, float q_scale) {
    float s[kBlock];
#pragma unroll
    for (int i = 0; i < kBlock; i += 32) tmem_ld32(s_tmem + i, s + i);
    tmem_ld_wait();
    float top = kNoScore;
#pragma unroll
    for (int g = 0; g < kBlock / 16; ++g) {
        float a = max3(s[g * 16], s[g * 16 + 1], s[g * 16 + 2]), b = max3(s[g * 16 + 3], s[g * 16 + 4], s[g * 16 + 5]);
#pragma unroll
        for (int i = 6; i < 14; i += 4) {
            a = max3(a, s[g * 16 + i], s[g * 16 + i + 1]);
            b = max3(b, s[g * 16 + i + 2], s[g * 16 + i + 3]);
        }
        a = max3(a, s[g * 16 + 14], s[g * 16 + 15]);
        top = fmaxf(top, fmaf(fmaxf(a, b), sc.key[g] * q_scale, sc.exponent[g]));
    }
    return top;
}
// Scores -> 2^(s f + exponent - m), whose sum without the exponents is returned, and times the values' weight as
// fp16 into the place of the scores.  A loop over 32 columns, read a second time, rather than 128 held and unrolled: the code of all
// six programs has to stay in the instruction caches.  The next columns are fetched as soon as the
// multiply-adds have taken these.
__device__ __forceinline__ float prompt_weights(uint32_t s_tmem, const PromptScales& sc, float q_scale, float m) {
    Pair sums[4] = {0, 0, 0, 0};                                    // independent: the additions must not wait for one another
    float s[32];
    tmem_ld32(s_tmem, s);
#pragma unroll 1
    for (int ch = 0; ch < 4; ++ch) {
        Pair e[16];
        const float f0 = sc.key[ch * 2] * q_scale, f1 = sc.key[ch * 2 + 1] * q_scale;
        const float c0 = sc.exponent[ch * 2] - m, c1 = sc.exponent[ch * 2 + 1] - m;
        const float w0 = sc.weight[ch * 2], w1 = sc.weight[ch * 2 + 1], b0 = sc.back[ch * 2], b1 = sc.back[ch * 2 + 1];
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i)
            e[i] = fma2(pair(s[2 * i], s[2 * i + 1]), i < 8 ? pair(f0, f0) : pair(f1, f1), i < 8 ? pair(c0, c0) : pair(c1, c1));
        tmem_ld32(s_tmem + (ch < 3 ? ch + 1 : 3) * 32, s);          // (the last time to no purpose: its columns are not written yet)
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            e[i] = pair(prompt_exp2(pair_x(e[i])), prompt_exp2(pair_y(e[i])));
            sums[i & 3] = fma2(e[i], i < 8 ? pair(b0, b0) : pair(b1, b1), sums[i & 3]);
            const Pair pw = mul2(e[i], i < 8 ? pair(w0, w0) : pair(w1, w1));
            const __half2 h = __floats2half2_rn(pair_x(pw), pair_y(pw));
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        tmem_st16(s_tmem + ch * 16, w);
    }
    tmem_ld_wait();
    const Pair sum = add2(add2(sums[0], sums[1]), add2(sums[2], sums[3]));
    return pair_x(sum) + pair_y(sum);
}
// The same for rows that see columns [lo, hi) only: at the diagonal, a window's edge or a sequence's end.  16
// columns at a time from tensor memory, to keep the code small.
__device__ __forceinline__ float prompt_top_seen(uint32_t s_tmem, const PromptScales& sc, float q_scale, int lo, int hi) {
    float top = kNoScore;
#pragma unroll 1
    for (int g = 0; g < kBlock / 16; ++g) {
        float s[16];
        tmem_ld16(s_tmem + g * 16, s);
        tmem_ld_wait();
        const uint32_t seen = prompt_seen(g * 16, lo, hi);
        float best = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) best = fmaxf(best, (seen >> i) & 1 ? s[i] : -INFINITY);
        top = fmaxf(top, fmaf(best, sc.key[g] * q_scale, sc.exponent[g]));
    }
    return top;
}
__device__ __forceinline__ float prompt_weights_seen(uint32_t s_tmem, const PromptScales& sc, float q_scale, float m, int lo, int hi) {
    float sum = 0.0f;
#pragma unroll 1
    for (int g = 0; g < kBlock / 16; ++g) {
        float s[16];
        tmem_ld16(s_tmem + g * 16, s);
        tmem_ld_wait();
        const uint32_t seen = prompt_seen(g * 16, lo, hi);
        const float f = sc.key[g] * q_scale, c = sc.exponent[g] - m, weight = sc.weight[g], back = sc.back[g];
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            // zero where the row does not see, not NaN from a scale that it does not see
            const bool a = (seen >> i) & 1, b = (seen >> (i + 1)) & 1;
            const float e0 = a ? prompt_exp2(fmaf(s[i], f, c)) : 0.0f, e1 = b ? prompt_exp2(fmaf(s[i + 1], f, c)) : 0.0f;
            sum = fmaf(e0 + e1, back, sum);
            const __half2 h = __floats2half2_rn(a ? e0 * weight : 0.0f, b ? e1 * weight : 0.0f);
            w[i / 2] = *reinterpret_cast<const uint32_t*>(&h);
        }
        tmem_st8(s_tmem + g * 8, w);
    }
    return sum;
}

template <int DIM, int FORMAT>
__global__ void __launch_bounds__(kPromptThreads, 1)
kv_prompt_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                 const __grid_constant__ PromptParams p) {
    using S = PromptShape<DIM>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t q_smem = smem, ring = q_smem + S::kQ, raw = ring + S::kRing * S::kTile;
    __shared__ PromptBars bars;
    __shared__ __align__(16) PromptScales scales[kScaleSlots];
    __shared__ int64_t scan[kPromptThreads / 32];
    __shared__ PromptPart parts[kPartSlots];
    __shared__ int abort_word;
    __shared__ uint32_t tmem_holder;

    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    if (t == 0) {
        for (int i = 0; i < 4; ++i) {
            mbar_init(smem_addr(&bars.raw_full[i]), 1);
            mbar_init(smem_addr(&bars.raw_empty[i]), 4);
            mbar_init(smem_addr(&bars.full[i]), 4);
            mbar_init(smem_addr(&bars.empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_addr(&bars.s_full[i]), 1);
            mbar_init(smem_addr(&bars.o_full[i]), 1);
            mbar_init(smem_addr(&bars.p_ready[i]), 4);
            mbar_init(smem_addr(&bars.q_full[i]), 4);
        }
        for (int i = 0; i < kScaleSlots; ++i) {
            mbar_init(smem_addr(&bars.scale_full[i]), 1);
            mbar_init(smem_addr(&bars.scale_empty[i]), 8);
        }
        for (int i = 0; i < kPartSlots; ++i) {
            mbar_init(smem_addr(&bars.part_full[i]), 1);
            mbar_init(smem_addr(&bars.part_empty[i]), 15);         // every warp but the one that writes them
        }
        mbar_init(smem_addr(&bars.drained), 1);
        abort_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kProductWarp) { tmem_alloc(smem_addr(&tmem_holder), 512); tmem_relinquish(); }

    // --- this CTA's share of the axis of key blocks
    const int per = (p.c.sequences + kPromptThreads - 1) / kPromptThreads;
    const int b0 = min(t * per, p.c.sequences), b1 = min(b0 + per, p.c.sequences);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) {
        PromptItem it;
        if (prompt_sequence(p, b, it)) mine += prompt_head_blocks(p, it) * p.c.kv_heads;
    }
    int64_t upto = mine;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, upto, x);
        if (lane >= x) upto += v;
    }
    if (lane == 31) scan[warp] = upto;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_holder;
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < kPromptThreads / 32; ++w) {
        if (w < warp) upto += scan[w];
        total += scan[w];
    }
    const int64_t ctas = min((int64_t)gridDim.x, total);
    const int64_t w0 = blockIdx.x < ctas ? total * blockIdx.x / ctas : total;
    const int64_t w1 = blockIdx.x < ctas ? total * (blockIdx.x + 1) / ctas : total;
    if (w0 < w1 && w0 >= upto - mine && w0 < upto) {               // exactly one thread
        int64_t rest = w0 - (upto - mine);
        PromptItem it;
        for (int b = b0; b < b1; ++b) {
            if (!prompt_sequence(p, b, it)) continue;
            const int64_t per_head = prompt_head_blocks(p, it);
            if (rest >= per_head * p.c.kv_heads) { rest -= per_head * p.c.kv_heads; continue; }
            it.kv_head = (int)(rest / per_head);
            rest -= it.kv_head * per_head;
            for (it.pair = 0;; ++it.pair) {
                prompt_range(p, it);
                if (rest < it.blocks + kItemCost) break;
                rest -= it.blocks + kItemCost;
            }
            break;
        }
        parts[0].it = it;
        parts[0].slot = 0;
        parts[0].set((int)rest, w1 - w0);
    }
    __syncthreads();
    int32_t* meta = p.meta + (int64_t)blockIdx.x * 8;
    if (t == 0) meta[0] = 0;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the joining kernel may take its place and wait

    if (w0 < w1) {
        volatile int* abort = &abort_word;
        uint32_t n_part = 0;
        // The next part of the list (the first is there from the start), and giving its slot back.
        auto part_wait = [&]() -> bool {
            return n_part == 0 || prompt_wait(smem_addr(&bars.part_full[n_part % kPartSlots]),
                                                    (n_part / kPartSlots) & 1, abort, wait_code(13, n_part % kPartSlots));
        };
        auto part_done = [&]() {
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_addr(&bars.part_empty[n_part % kPartSlots]));
            ++n_part;
        };

        if (warp < kConvertWarp) {
            // ------------------------------------------------------------------ softmax
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
            const int tile = warp >> 2, row = (warp & 3) * 32 + lane;
            const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
            const uint32_t s_tmem = tmem + tile * 128 + lanes, o_tmem = tmem + S::kO + tile * DIM + lanes;
            const int row_token = row / p.head_tile, row_head = row - row_token * p.head_tile;
            uint32_t blocks_seen = 0, scale_uses = 0, o_uses = 0;
            bool ok = true, more = true;

            // This row's query to shared memory as fp16 times a power of two; returns what the scores are times.
            auto load_q = [&](const PromptItem& it) -> float {
                const int tok = it.token0 + tile * p.token_tile + row_token, hd = it.head0 + row_head;
                const bool there = row_token < p.token_tile && tok < it.count && hd < p.a.group;
                const int64_t at = (it.begin + tok) * p.a.q_token_stride + ((int64_t)it.kv_head * p.a.group + hd) * p.a.q_head_stride;
                const uint16_t* q = static_cast<const uint16_t*>(p.a.q) + at;
                const bool vector = (reinterpret_cast<uintptr_t>(q) & 15) == 0;
                // the whole row at once: its latency, not its bytes, is what counts between two parts
                uint32_t w[DIM / 2];
#pragma unroll
                for (int c = 0; c < DIM / 8; ++c) {
                    uint4 x = make_uint4(0, 0, 0, 0);
                    if (there && vector && c * 8 < p.c.head_dim) x = *reinterpret_cast<const uint4*>(q + c * 8);
                    w[c * 4] = x.x; w[c * 4 + 1] = x.y; w[c * 4 + 2] = x.z; w[c * 4 + 3] = x.w;
                }
                if (there && !vector) {
#pragma unroll
                    for (int i = 0; i < DIM / 2; ++i)
                        if (2 * i < p.c.head_dim) w[i] = q[2 * i] | (uint32_t)q[2 * i + 1] << 16;
                }
                // magnitudes order like their bits in either type
                uint32_t size = 0;
#pragma unroll
                for (int i = 0; i < DIM / 2; ++i) size = max(size, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
                const float largest = p.a.type == RNS_F16 ? __half2float(__ushort_as_half((uint16_t)size))
                                                          : __uint_as_float(size << 16);
                const uint32_t bits = __float_as_uint(largest);
                const int e = (int)(bits >> 23);
                const int shift = bits == 0 || e == 255 ? 0 : max(-126, min(120, 134 - e));
                const float up = __uint_as_float((uint32_t)(shift + 127) << 23) * p.sign;
                const float down = __uint_as_float((uint32_t)(127 - max(-120, min(126, shift))) << 23);
#pragma unroll
                for (int c = 0; c < DIM / 8; ++c) {
                    float v[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t x = w[c * 4 + i];
                        if (p.a.type == RNS_F16) {
                            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x));
                            v[2 * i] = f.x; v[2 * i + 1] = f.y;
                        } else {
                            v[2 * i] = __uint_as_float(x << 16); v[2 * i + 1] = __uint_as_float(x & 0xffff0000u);
                        }
                    }
                    uint32_t h[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        // int8 tiles hold dimensions 0 2 1 3 of every four
                        const int a = FORMAT == RNS_KV_INT8 ? (i >> 1) * 4 + (i & 1) : 2 * i;
                        const int b = FORMAT == RNS_KV_INT8 ? a + 2 : a + 1;
                        const __half2 f = __floats2half2_rn(v[a] * up, v[b] * up);
                        h[i] = *reinterpret_cast<const uint32_t*>(&f);
                    }
                    const uint32_t to = q_smem + tile * S::kQTile + (c >> 3) * (kTileRows * 128) + row * 128 +
                                        (((c & 7) ^ (row & 7)) << 4);
                    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(to), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_addr(&bars.q_full[tile]));
                return p.a.scale_log2 * p.sign * down;
            };

            float q_scale = parts[0].mine1[tile] > parts[0].mine0[tile] ? load_q(parts[0].it) : 0.0f;
            while (more && ok) {
                const PromptPart& part = parts[n_part % kPartSlots];
                const PromptItem& it = part.it;
                const int mine0 = part.mine0[tile], mine1 = part.mine1[tile], live1 = part.live1, key0 = it.key0;
                const int tok = it.token0 + tile * p.token_tile + row_token;
                const int position = it.length - it.count + tok;
                const int hi = position < 0 ? 0 : p.a.causal ? position + 1 : it.length;
                const int lo = kv_first_key(p.a, position);
                // keys that every row of the tile sees
                const int tile_pos = it.length - it.count + it.token0 + tile * p.token_tile;
                const int all_hi = p.a.causal ? tile_pos + 1 : tile_pos >= 0 ? it.length : 0;
                const int all_lo = kv_first_key(p.a, tile_pos + p.token_tile - 1);
                float m = kNoScore, l = 0.0f;
                for (int j = part.live0; j < live1; ++j) {
                    const int slot = scale_uses % kScaleSlots;
                    ok = prompt_wait(smem_addr(&bars.scale_full[slot]), (scale_uses / kScaleSlots) & 1, abort, wait_code(1, slot));
                    ++scale_uses;
                    if (!ok) break;
                    if (j < mine0 || j >= mine1) {
                        if (lane == 0) mbar_arrive(smem_addr(&bars.scale_empty[slot]));
                        continue;
                    }
                    const PromptScales& sc = scales[slot];
                    ok = prompt_wait(smem_addr(&bars.s_full[tile]), blocks_seen & 1, abort, wait_code(2, tile));
                    if (!ok) break;
                    ++blocks_seen;
                    tc_fence_after();
                    const int key = key0 + j * kBlock;
                    const bool whole = key + kBlock <= all_hi && key >= all_lo;
                    float top = whole ? prompt_top(s_tmem, sc, q_scale) : prompt_top_seen(s_tmem, sc, q_scale, lo - key, hi - key);
                    if (__any_sync(0xffffffffu, top > m + kScoreLag)) {
                        top = top > m + kScoreLag ? ceilf(top) : m;
                        const float keep = prompt_exp2(m - top);
                        m = top;
                        l *= keep;
                        // S(j) has arrived, so the product of the block before has: O is at rest
                        if (j > mine0) {
#pragma unroll 1
                            for (int ch = 0; ch < DIM / 8; ++ch) {
                                float o[8];
                                uint32_t v[8];
                                tmem_ld8f(o_tmem + ch * 8, o);
                                tmem_ld_wait();
#pragma unroll
                                for (int i = 0; i < 8; ++i) v[i] = __float_as_uint(o[i] * keep);
                                tmem_st8(o_tmem + ch * 8, v);
                            }
                        }
                    }
                    l += whole ? prompt_weights(s_tmem, sc, q_scale, m) : prompt_weights_seen(s_tmem, sc, q_scale, m, lo - key, hi - key);
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(smem_addr(&bars.p_ready[tile]));
                        mbar_arrive(smem_addr(&bars.scale_empty[slot]));
                    }
                }
                if (!ok) break;
                // the next part's queries before this one's output: their products can start meanwhile
                more = !part.last;
                float next_scale = 0.0f;
                if (more) {
                    ++n_part;
                    ok = part_wait();
                    const PromptPart& next = parts[n_part % kPartSlots];
                    if (ok && next.mine1[tile] > next.mine0[tile]) next_scale = load_q(next.it);
                    --n_part;
                    if (!ok) break;
                }
                const bool any = mine1 > mine0;
                if (any) {
                    ok = prompt_wait(smem_addr(&bars.o_full[tile]), o_uses & 1, abort, wait_code(3, tile));
                    ++o_uses;
                    if (!ok) break;
                    tc_fence_after();
                }
                // the row's output: to its place, or as a piece of it (largest score, sum, O) to the workspace
                const bool complete = part.step == 0 && part.stop == it.blocks, empty = m == kNoScore && l == 0.0f;
                const bool there = tile < S::kTiles && row_token < p.token_tile && it.token0 + tile * p.token_tile + row_token < it.count &&
                                   it.head0 + row_head < p.a.group;
                const int64_t token = it.begin + it.token0 + tile * p.token_tile + row_token;
                const int64_t head = (int64_t)it.kv_head * p.a.group + it.head0 + row_head;
                const bool none = part.stop == part.step;
                float* piece = p.partial + ((int64_t)blockIdx.x * 2 + part.slot) * S::kPartial;
                const int at = tile * kTileRows + row;
                const float factor = complete ? (empty ? 0.0f : 1.0f / l) : 1.0f;
#pragma unroll 1
                for (int d = 0; d < DIM && !none; d += 16) {
                    float o[16];
                    if (any) {
                        tmem_ld16(o_tmem + d, o);
                        tmem_ld_wait();
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = any ? o[i] * factor : 0.0f;
                    if (FORMAT == RNS_KV_INT8) {                    // columns hold dimensions 0 2 1 3 of every four
#pragma unroll
                        for (int i = 0; i < 16; i += 4) { const float x = o[i + 1]; o[i + 1] = o[i + 2]; o[i + 2] = x; }
                    }
                    if (!complete) {
                        float4* to = reinterpret_cast<float4*>(piece + 4 * kTileRows + at * DIM + d);
#pragma unroll
                        for (int i = 0; i < 4; ++i) to[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    } else if (there && d < p.c.head_dim) {
                        uint32_t h[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            if (p.a.type == RNS_F16) {
                                const __half2 f = __floats2half2_rn(o[2 * i], o[2 * i + 1]);
                                h[i] = *reinterpret_cast<const uint32_t*>(&f);
                            } else {
                                const __nv_bfloat162 f = __floats2bfloat162_rn(o[2 * i], o[2 * i + 1]);
                                h[i] = *reinterpret_cast<const uint32_t*>(&f);
                            }
                        }
                        uint16_t* out = static_cast<uint16_t*>(p.a.out) + token * p.a.out_token_stride + head * p.a.out_head_stride + d;
                        if ((reinterpret_cast<uintptr_t>(out) & 15) == 0) {
                            reinterpret_cast<uint4*>(out)[0] = make_uint4(h[0], h[1], h[2], h[3]);
                            reinterpret_cast<uint4*>(out)[1] = make_uint4(h[4], h[5], h[6], h[7]);
                        } else {
#pragma unroll
                            for (int e = 0; e < 16; ++e) out[e] = (uint16_t)(h[e / 2] >> (16 * (e & 1)));
                        }
                    }
                }
                if (none) {
                    // not a block of this item: the next CTA starts it
                } else if (complete) {
                    if (p.a.lse != nullptr && there)
                        p.a.lse[token * p.a.heads + head] = empty ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
                } else {
                    piece[at] = m;
                    piece[2 * kTileRows + at] = l;
                    if (part.step == 0 && t == 0) {
                        // this CTA holds the first piece: it names the item and where its pieces are
                        const int64_t end = w1 - part.left - part.at + it.blocks + kItemCost;
                        int64_t last = (end - 1) * ctas / total;
                        while (total * (last + 1) / ctas < end) ++last;
                        while (total * last / ctas > end - 1) --last;
                        meta[1] = (int)(last - blockIdx.x) + 1;
                        meta[2] = part.slot;
                        meta[3] = it.b; meta[4] = it.kv_head; meta[5] = it.token0; meta[6] = it.head0;
                        meta[0] = 1;
                    }
                }
                if (any) tc_fence_before();
                q_scale = next_scale;
                part_done();
            }
        } else {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        }
        if (warp >= kConvertWarp && warp < kProductWarp) {
            // ------------------------------------------------------------------ 8-bit tiles -> fp16 tiles
            const int lane_key = ((lane >> 3) & 3) ^ (((lane >> 2) & 1) * 5), lane_chunk = lane & 3;
            // byte of this lane's chunk in 8 keys as TMA swizzled them, and of its two chunks in a part of the fp16 tile
            const uint32_t raw_at = DIM == 64 ? lane_key * 64 + ((lane_chunk ^ ((lane_key >> 1) & 3)) << 4)
                                              : lane_key * 128 + ((lane_chunk ^ (lane_key & 3)) << 4);
            const uint32_t raw_flip = (lane_key & 4) << 4, out0 = ((2 * lane_chunk) ^ lane_key) << 4;
            uint32_t n = 0;
            bool ok = true, more = true;
            while (more && (ok = ok && part_wait())) {
                const PromptPart& part = parts[n_part % kPartSlots];
                more = !part.last;
                const int live1 = part.live1, tokens = part.it.length - part.it.key0;
                for (int j = part.live0; j < live1 && ok; ++j) {
                    const int valid = tokens - j * kBlock;                                // rows with a token
#pragma unroll 1
                    for (int side = 0; side < 2; ++side, ++n) {
                        const int rs = n % S::kRawRing, slot = n % S::kRing;
                        ok = prompt_wait(smem_addr(&bars.raw_full[rs]), (n / S::kRawRing) & 1, abort, wait_code(4, rs)) &&
                             prompt_wait(smem_addr(&bars.empty[slot]), ((n / S::kRing) & 1) ^ 1, abort, wait_code(5, slot));
                        if (!ok) break;
                        const uint32_t from = raw + rs * S::kRaw, to = ring + slot * S::kTile;
                        // Units of 8 keys x 64 dimensions, one 16-byte chunk a lane.  Eight neighbouring lanes hold
                        // four chunks of keys k and k ^ 5, whose swizzles differ in bits 0 and 2: neither the
                        // 16-byte loads nor the stores meet a bank twice, and every swizzle is a constant of the lane.
#pragma unroll 2
                        for (int u = warp - kConvertWarp; u < kBlock / 8 * S::kParts; u += 4) {
                            const int part64 = u % S::kParts, keys = u / S::kParts * 8;
                            const uint32_t at = DIM == 64 ? from + keys * 64 + raw_at
                                                          : from + (part64 >> 1) * (kBlock * 128) + keys * 128 + raw_at + ((part64 & 1) << 6 ^ raw_flip);
                            uint32_t w[4];
                            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at));
                            // bytes behind the sequence may be NaN patterns, which no weight of zero removes
                            if (FORMAT == RNS_KV_E4M3 && keys + lane_key >= valid) w[0] = w[1] = w[2] = w[3] = 0;
                            uint32_t h[8];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                if (FORMAT == RNS_KV_INT8) { h[2 * k] = half_pair_s8(w[k]); h[2 * k + 1] = half_pair_s8(w[k] >> 8); }
                                else { h[2 * k] = half_pair_e4m3(w[k]); h[2 * k + 1] = half_pair_e4m3(w[k] >> 16); }
                            }
                            const uint32_t out = to + part64 * (kBlock * 128) + keys * 128 + lane_key * 128;
                            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(out + out0), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
                            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(out + (out0 ^ 16)), "r"(h[4]), "r"(h[5]), "r"(h[6]), "r"(h[7]) : "memory");
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(smem_addr(&bars.raw_empty[rs]));
                            mbar_arrive(smem_addr(&bars.full[slot]));
                        }
                    }
                }
                part_done();
            }
        } else if (warp == kProductWarp) {
            // ------------------------------------------------------------------ products
            // The whole warp walks along and one elected lane issues: descriptors are then uniform values,
            // which the instruction takes from uniform registers (from one lane's registers each product
            // cost over 250 cycles to issue).
            const uint32_t idesc_s = f16_idesc(128, kBlock, false), idesc_o = f16_idesc(128, DIM, true);
            uint32_t n = 0, q_uses[2] = {0, 0}, p_uses = 0;              // p_uses: a phase bit for each tile
            bool ok = true, more = true;
            const auto uniform = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
            const uint32_t tm = uniform(tmem);
            auto wait = [&](uint64_t& bar, uint32_t parity, int role, int index) {
                if (ok) ok = prompt_wait(smem_addr(&bar), parity & 1, abort, wait_code(role, index));
                tc_fence_after();
            };
            while (more && (ok = ok && part_wait())) {
                const PromptPart& part = parts[n_part % kPartSlots];
                more = !part.last;
                const int live0 = uniform(part.live0), live1 = uniform(part.live1);
                const int from0 = uniform(part.mine0[0]), to0 = uniform(part.mine1[0]);
                const int from1 = uniform(part.mine0[1]), to1 = uniform(part.mine1[1]);
                if (to0 > from0) wait(bars.q_full[0], q_uses[0]++, 6, 0);
                if (to1 > from1) wait(bars.q_full[1], q_uses[1]++, 6, 1);
                // Block j's second product, then block j + 1's first into the same columns, tile after tile.
                // n counts tiles: keys of block j at n, its values at n + 1, the next keys at n + 2.
                const uint64_t q0 = make_smem_desc(q_smem, 128);
#pragma unroll 1
                for (int j = live0 - 1; j < live1 && live0 < live1; ++j) {
                    const bool now = j >= live0, again = j + 1 < live1;
                    const uint32_t k_index = now ? n + 2 : n, k_slot = k_index % S::kRing, v_slot = (n + 1) % S::kRing;
                    // tiles are converted in order: the next keys are there after these values
                    if (again) wait(bars.full[k_slot], k_index / S::kRing, 7, k_slot);
                    else wait(bars.full[v_slot], (n + 1) / S::kRing, 8, v_slot);
                    const uint64_t k_desc = make_smem_desc(ring + k_slot * S::kTile, 128);
                    const uint64_t v_desc = mn_desc(ring + v_slot * S::kTile, kBlock * 128, 1024);
#pragma unroll 1
                    for (int tile = 0; tile < 2 && ok; ++tile) {
                        const int from = tile ? from1 : from0, to = tile ? to1 : to0;
                        const bool second = j >= from && j < to, first = again && j + 1 >= from && j + 1 < to;
                        if (second) {
                            wait(bars.p_ready[tile], p_uses >> (tile * 8), 9, tile);
                            p_uses ^= 1u << (tile * 8);
                            if (!ok) break;
                        }
                        const uint32_t s_d = tm + tile * 128, o_d = tm + S::kO + tile * DIM;
                        const uint64_t q_desc = q0 + tile * (S::kQTile >> 4);
                        if (elect_one()) {
                            if (second) {
#pragma unroll
                                for (int k = 0; k < kBlock / 16; ++k)
                                    umma_f16_ts(o_d, s_d + k * 8, v_desc + (k * 2048 >> 4), idesc_o, k > 0 || j > from);
                                if (j + 1 == to) umma_commit(smem_addr(&bars.o_full[tile]));
                            }
                            if (first) {
#pragma unroll
                                for (int k = 0; k < DIM / 16; ++k) {
                                    const uint32_t off = ((k >> 2) * (128 * 128) + (k & 3) * 32) >> 4;
                                    umma_f16(s_d, q_desc + off, k_desc + off, idesc_s, k > 0);
                                }
                                umma_commit(smem_addr(&bars.s_full[tile]));
                            }
                            if (tile == 1) {
                                if (now) umma_commit(smem_addr(&bars.empty[v_slot]));
                                if (again) umma_commit(smem_addr(&bars.empty[k_slot]));
                            }
                        }
                        __syncwarp();
                    }
                    if (!ok) break;
                    if (now) n += 2;
                }
                if (ok) part_done();
            }
            // nothing may still be on its way to this CTA's barriers when it leaves
            for (uint32_t i = n > S::kRing ? n - S::kRing : 0; i < n && ok; ++i)
                wait(bars.empty[i % S::kRing], i / S::kRing, 10, i % S::kRing);
            if (!ok) {                                             // nor read and write memory that is given back
                if (elect_one()) umma_commit(smem_addr(&bars.drained));
                __syncwarp();
                prompt_drain(smem_addr(&bars.drained), 0);
            }
        } else if (warp == kCopyWarp) {
            // ------------------------------------------------------------------ copies
            uint32_t n = 0;
            bool ok = true, more = true;
            const int boxes = kBlock / p.box_rows;
            while (more && (ok = ok && part_wait())) {
                const PromptPart& part = parts[n_part % kPartSlots];
                more = !part.last;
                const int live1 = part.live1, b = part.it.b, kv_head = part.it.kv_head, key0 = part.it.key0, length = part.it.length;
                // Page indices of four blocks at a time, eight lanes a block, and those of the next four while
                // these are copied: one after the other, their latency was most of a block's time.
                const int live0 = part.live0, box = lane & 7;
                const auto entry = [&](int at) {
                    const int key = key0 + (at + (lane >> 3)) * kBlock + box * p.box_rows;
                    return at + (lane >> 3) < live1 && box < boxes && key < length ? kv_entry(p.c, b, key >> p.c.page_shift) : -1;
                };
                int32_t next = entry(live0);
                for (int j0 = live0; j0 < live1 && ok; j0 += 4) {
                    const int32_t named = next;
                    next = entry(j0 + 4);
                    const int key = key0 + (j0 + (lane >> 3)) * kBlock + box * p.box_rows;
                    int z = (int)p.c.pages;                            // behind the last page: zeros
                    if (j0 + (lane >> 3) < live1 && box < boxes && key < length) {
                        const int page = kv_named(p.c, named);
                        if (page >= 0) z = page;
                    }
#pragma unroll 1
                    for (int u = 0; u < 8 && j0 + (u >> 1) < live1; ++u, ++n) {
                        const int rs = n % S::kRawRing, side = u & 1;
                        ok = prompt_wait(smem_addr(&bars.raw_empty[rs]), ((n / S::kRawRing) & 1) ^ 1, abort, wait_code(11, rs));
                        if (!ok) break;
                        const uint32_t bar = smem_addr(&bars.raw_full[rs]);
                        if (lane == 0) mbar_arrive_expect_tx(bar, S::kRaw);
                        __syncwarp();
                        if ((lane >> 3) == (u >> 1) && box < boxes) {
                            const uint32_t to = raw + rs * S::kRaw + box * p.box_rows * (DIM == 64 ? 64 : 128);
                            const int y = kv_head * p.c.page_tokens + (key & (p.c.page_tokens - 1));
                            tma_load_3d(to, side ? &map_v : &map_k, bar, 0, y, z);
                            if (DIM == 256) tma_load_3d(to + kBlock * 128, side ? &map_v : &map_k, bar, 128, y, z);
                        }
                    }
                }
                part_done();
            }
            for (uint32_t i = n > S::kRawRing ? n - S::kRawRing : 0; i < n; ++i)
                prompt_drain(smem_addr(&bars.raw_full[i % S::kRawRing]), (i / S::kRawRing) & 1);
        } else if (warp == kScaleWarp) {
            // ------------------------------------------------------------------ scales of the pages
            uint32_t n = 0;
            bool ok = true, more = true;
            while (more && (ok = ok && part_wait())) {
                const PromptPart& part = parts[n_part % kPartSlots];
                more = !part.last;
                const int live1 = part.live1, b = part.it.b, kv_head = part.it.kv_head, key0 = part.it.key0;
                const int length = part.it.length;
                // four blocks at a time, as the copies: a lane for 16 keys
                const int live0 = part.live0, mine = lane >> 3;
                const auto entry = [&](int at) {
                    const int key = key0 + (at + mine) * kBlock + (lane & 7) * 16;
                    return at + mine < live1 && key < length ? kv_entry(p.c, b, key >> p.c.page_shift) : -1;
                };
                int32_t next = entry(live0);
                for (int j0 = live0; j0 < live1 && ok; j0 += 4) {
                    const int32_t named = next;
                    const int key = key0 + (j0 + mine) * kBlock + (lane & 7) * 16;
                    float ks = 0.0f, vs = 0.0f;
                    if (j0 + mine < live1 && key < length) {
                        const int page = kv_named(p.c, named);
                        if (page >= 0) {
                            const int64_t block = (int64_t)page * p.c.kv_heads + kv_head;
                            ks = p.c.scale[0][block];
                            vs = p.c.scale[1][block];
                        }
                    }
                    next = entry(j0 + 4);
                    const KvValueScale value = kv_value_scale(vs);
#pragma unroll 1
                    for (int i = 0; i < 4 && j0 + i < live1; ++i) {
                        const int slot = n % kScaleSlots;
                        ok = prompt_wait(smem_addr(&bars.scale_empty[slot]), ((n / kScaleSlots) & 1) ^ 1, abort, wait_code(12, slot));
                        if (!ok) break;
                        ++n;
                        if (mine == i) {
                            scales[slot].key[lane & 7] = ks;
                            scales[slot].exponent[lane & 7] = value.exponent;
                            scales[slot].weight[lane & 7] = value.weight;
                            scales[slot].back[lane & 7] = value.back;
                        }
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_addr(&bars.scale_full[slot]));
                    }
                }
                part_done();
            }
        } else if (warp == kPartWarp) {
            // ------------------------------------------------------------------ parts
            PromptPart part = parts[0];
            bool ok = true;
            if (lane == 0) mbar_arrive(smem_addr(&bars.part_full[0]));      // keeps slot 0's phases in step
            for (uint32_t n = 1; ok && !part.last; ++n) {
                prompt_next(p, part);
                const int slot = n % kPartSlots;
                ok = prompt_wait(smem_addr(&bars.part_empty[slot]), ((n / kPartSlots) & 1) ^ 1, abort, wait_code(14, slot));
                if (!ok) break;
                if (lane == 0) {
                    parts[slot] = part;
                    mbar_arrive(smem_addr(&bars.part_full[slot]));
                }
                __syncwarp();
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kProductWarp) tmem_dealloc(tmem, 512);
    if (abort_word != 0 && t == 0 && p.c.status != nullptr) *p.c.status = RNS_ERR_DEVICE_TIMEOUT;
}

// Joins the pieces of the items that a CTA boundary cut: block (first piece's CTA, 8 rows), a warp a row.
template <int DIM>
__global__ void __launch_bounds__(256) kv_prompt_join_kernel(const __grid_constant__ PromptParams p) {
    using S = PromptShape<DIM>;
    asm volatile("griddepcontrol.wait;" ::: "memory");             // the pieces are complete and visible
    const int32_t* meta = p.meta + (int64_t)blockIdx.x * 8;
    if (meta[0] == 0) return;
    const int lane = threadIdx.x & 31, at = blockIdx.y * 8 + (threadIdx.x >> 5);
    const int tile = at / kTileRows, row = at % kTileRows;
    const int row_token = row / p.head_tile, row_head = row - row_token * p.head_tile;
    const KvSpan s = kv_span(p.c, p.a.lens, p.a.starts, p.a.tokens, meta[3]);
    const int tok = meta[5] + tile * p.token_tile + row_token, hd = meta[6] + row_head;
    if (tile >= S::kTiles || row_token >= p.token_tile || tok >= s.count || hd >= p.a.group) return;
    const int pieces = meta[1];
    const float* first = p.partial + ((int64_t)blockIdx.x * 2 + meta[2]) * S::kPartial;
    const float* next = p.partial + ((int64_t)blockIdx.x + 1) * 2 * S::kPartial;
    const auto piece = [&](int i) { return i == 0 ? first : next + (int64_t)(i - 1) * 2 * S::kPartial; };
    float top = kNoScore;
    for (int i = lane; i < pieces; i += 32) top = fmaxf(top, piece(i)[at]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    float sum = 0.0f, o[DIM / 32] = {};
    for (int base = 0; base < pieces; base += 32) {                // pieces in key order, their loads in flight together
        float mine = 0.0f, total = 0.0f;
        if (base + lane < pieces) {
            mine = prompt_exp2(piece(base + lane)[at] - top);
            total = piece(base + lane)[2 * kTileRows + at];
        }
        const int n = min(32, pieces - base);
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
            const float* part = piece(base + i) + 4 * kTileRows + at * DIM + lane;
            const float f = __shfl_sync(0xffffffffu, mine, i);
            sum = fmaf(__shfl_sync(0xffffffffu, total, i), f, sum);
#pragma unroll
            for (int j = 0; j < DIM / 32; ++j) o[j] = fmaf(part[j * 32], f, o[j]);
        }
    }
    const bool empty = top == kNoScore && sum == 0.0f;
    const float inv = empty ? 0.0f : 1.0f / sum;
    const int64_t token = s.begin + tok, head = (int64_t)meta[4] * p.a.group + hd;
#pragma unroll
    for (int j = 0; j < DIM / 32; ++j) {
        const int d = j * 32 + lane;
        if (d >= p.c.head_dim) continue;
        const int64_t to = token * p.a.out_token_stride + head * p.a.out_head_stride + d;
        if (p.a.type == RNS_F16) static_cast<__half*>(p.a.out)[to] = __float2half_rn(o[j] * inv);
        else static_cast<__nv_bfloat16*>(p.a.out)[to] = __float2bfloat16_rn(o[j] * inv);
    }
    if (p.a.lse != nullptr && lane == 0)
        p.a.lse[token * p.a.heads + head] = empty ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int64_t kv_prompt_workspace(const KvView& c) {
    int sms = 0;
    if (sm_count(&sms) != RNS_OK) return -RNS_ERR_CUDA;
    const int piece = c.head_dim <= 64 ? PromptShape<64>::kPartial : c.head_dim <= 128 ? PromptShape<128>::kPartial : PromptShape<256>::kPartial;
    return (int64_t)sms * (2 * piece * 4 + 32);
}

template <int DIM, int FORMAT> static int launch_prompt(PromptParams& p, void* workspace, cudaStream_t st) {
    using S = PromptShape<DIM>;
    static_assert(S::kSmem + 2048 <= 227 * 1024, "one CTA per SM");
    int sms = 0;
    if (int rc = sm_count(&sms)) return rc;
    p.box_rows = p.c.page_tokens;
    p.tiles = S::kTiles;
    CUtensorMap maps[2];
    for (int i = 0; i < 2; ++i) {
        const uint64_t dims[3] = {(uint64_t)p.c.head_dim, (uint64_t)p.c.kv_heads * p.c.page_tokens, (uint64_t)p.c.pages};
        const uint64_t strides[2] = {dims[0], dims[0] * dims[1]};
        const uint32_t box[3] = {DIM == 64 ? 64u : 128u, (uint32_t)p.box_rows, 1u};
        if (int rc = make_map(&maps[i], p.c.data[i], 3, dims, strides, box, DIM == 64 ? 64 : 128)) return rc;
    }
    p.meta = static_cast<int32_t*>(workspace);
    p.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + (int64_t)sms * 32);
    const auto kernel = kv_prompt_kernel<DIM, FORMAT>;
    // a library that was built some other way: the split of the registers counts on this launch (looked up once)
    static const int regs = [&] { cudaFuncAttributes a; return cudaFuncGetAttributes(&a, kernel) == cudaSuccess ? a.numRegs : 0; }();
    if (regs < kLaunchRegs) return fail(RNS_ERR_UNSUPPORTED, "the prompt kernel was built with %d registers, not %d", regs, kLaunchRegs);
    static std::atomic<uint64_t> allowed{0};
    if (int rc = allow_smem(reinterpret_cast<const void*>(kernel), S::kSmem, &allowed)) return rc;
    kernel<<<sms, kPromptThreads, S::kSmem, st>>>(maps[0], maps[1], p);
    RNS_CUDA_OK(cudaGetLastError());
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)sms, 2 * kTileRows / 8);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    RNS_CUDA_OK(cudaLaunchKernelEx(&cfg, kv_prompt_join_kernel<DIM>, p));
    return RNS_OK;
}

int kv_prompt(const KvView& c, const KvQuery& a, int format, int min_rows_tokens, void* workspace, cudaStream_t st) {
    PromptParams p;
    memset(&p, 0, sizeof(p));
    p.c = c; p.a = a;
    p.min_rows_tokens = min_rows_tokens;
    p.sign = a.scale_log2 < 0.0f ? -1.0f : 1.0f;
    p.head_tile = a.group < kTileRows ? a.group : kTileRows;
    p.token_tile = kTileRows / p.head_tile;
    p.head_tiles = (a.group + p.head_tile - 1) / p.head_tile;
    if (c.head_dim <= 64)
        return format == RNS_KV_INT8 ? launch_prompt<64, RNS_KV_INT8>(p, workspace, st) : launch_prompt<64, RNS_KV_E4M3>(p, workspace, st);
    if (c.head_dim <= 128)
        return format == RNS_KV_INT8 ? launch_prompt<128, RNS_KV_INT8>(p, workspace, st) : launch_prompt<128, RNS_KV_E4M3>(p, workspace, st);
    return format == RNS_KV_INT8 ? launch_prompt<256, RNS_KV_INT8>(p, workspace, st) : launch_prompt<256, RNS_KV_E4M3>(p, workspace, st);
}

}  // namespace rns

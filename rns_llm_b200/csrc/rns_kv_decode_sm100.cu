// Attention of a few query rows per sequence over the paged 8-bit cache (decode steps, verification
// of drafted tokens).
//
// The rows of a tile are the queries that share a head of the cache: `group` heads of up to a few
// tokens.  With so few rows every cached byte is used once or a few times, so the bound is reading
// the cache.  What follows from that:
//
// * Work is cut along the keys.  All (sequence, head, row tile) items and their key steps form one
//   axis; each CTA takes an equal share of it, whatever the lengths are (they are only known on the
//   device).  A CTA that ends inside an item leaves the running maximum, sum and unnormalised output
//   in the workspace, and a second small kernel joins the pieces in key order.
// * A warp owns every fourth group of kKeys keys of its CTA's share and keeps a ring of such groups
//   in flight with TMA copies of its own, together with the pages' scales; the four warps meet only
//   at the end of an item.
// * Keys are the M operand of the first product (S^T = K Q^T) and values the M operand of the second
//   (O^T = V^T P^T), so that eight query rows fill the N = 8 of mma.sync.m16n8k16; tcgen05 needs 128
//   rows of M on the query side or twice the passes over shared memory.  Bytes become fp16 on the way
//   from shared memory to registers - int8 by setting the exponent of 1024 + 128 and one packed
//   subtraction, exact; e4m3 with the conversion instruction, exact - in whatever order of the inner
//   index costs least: sums do not depend on it, and Q is laid out to match.
// * Queries are scaled by a power of two per row into fp16's range, exact for bf16 as well up to
//   2^-32 of the row's largest element.  Scores, the softmax and all sums are fp32.  Each weight, with
//   its page's value scale, meets the values as two fp16 numbers, itself rounded and what that left
//   (2^-22), in units of a power of two near the row's largest such weight (kv_value_scale); the
//   accumulators need no scale of their own.  Small weights are off by up to 2^-25 of the unit each.
//   Rounded once, outputs in fp16 were off by 0.0003 where rounding the exact result gives 0.0002; the
//   second part costs 2 to 4 % (64 sequences 142.5 -> 145.5 us, one of 131072 tokens 65.8 -> 68.6; a
//   branch that leaves it out for bf16, whose own rounding hides it, costs as much: 145.0, 68.1).
// * The running maximum may lag by 2^8: then weights exceed one but nothing is lost, and the
//   accumulators are rescaled only when a vote finds a larger score.  It is a whole number, so that
//   rescaling is exact, and follows the row's own scores and their pages' scales alone: what a row
//   gives does not depend on the rows beside it.
//
// Measured (graph replay): 64 sequences of 1..8192 tokens, 32 over 8 heads of 128, 145 us = 3.7 TB/s of cache
// (0.57 of the copy rate; about 470 instructions for 16 keys, issue slots 53 % busy with three warps a scheduler: the
// latency of dependent instructions bounds it); one sequence of 131072, e4m3, 70 us; 8 of 640, 12 heads of 64, 16 us.
#include "rns_kv.cuh"
#include "rns_ptx.cuh"

namespace rns {

constexpr int kDecodeWarps = 4;
constexpr int kDecodeMostCtas = 3;      // of an SM
constexpr int kDecodeThreads = kDecodeWarps * 32;
constexpr float kNoMax = -1.7e38f;      // below every score: "nothing seen yet"
constexpr float kLag = 8.0f;            // how far a score may exceed the running maximum (log2)

struct DecodeParams {
    KvView c;
    KvQuery a;
    int head_tile, token_tile;          // rows of a tile: token_tile tokens x head_tile heads
    int head_tiles;                     // ceil(group / head_tile)
    int max_rows_tokens;                // sequences with more new tokens are left to the other kernel
    float* partial;                     // [grid][2][rows * (2 + DIM)]
    int32_t* meta;                      // [grid][8]
};

// One row tile of one sequence and head, and the keys it needs.
struct DecodeItem {
    int b, kv_head, tile;               // tile = token tile * head_tiles + head tile
    int64_t begin;
    int count, length;
    int key0, last, steps;              // first key (a multiple of the step's granule), end, key steps
};

template <int STEP, int KEYS>
__device__ __forceinline__ void decode_range(const DecodeParams& p, DecodeItem& it) {
    const int t0 = it.tile / p.head_tiles * p.token_tile, t1 = min(t0 + p.token_tile, it.count);
    const int base = it.length - it.count;
    int last = p.a.causal ? base + t1 : it.length;
    const int first = max(0, kv_first_key(p.a, base + t0));
    if (base + t1 <= 0) last = 0;
    it.key0 = first & ~(KEYS - 1);
    it.last = last;
    it.steps = last > it.key0 ? (last - it.key0 + STEP - 1) / STEP : 0;
    // a tile that sees nothing still has its zeros to write
    if (it.steps <= 0) it.steps = 1;
}
__device__ __forceinline__ int decode_tiles(const DecodeParams& p, int count) {
    return (count + p.token_tile - 1) / p.token_tile * p.head_tiles;
}
__device__ __forceinline__ bool decode_sequence(const DecodeParams& p, int b, DecodeItem& it) {
    const KvSpan s = kv_span(p.c, p.a.lens, p.a.starts, p.a.tokens, b);
    it.b = b; it.begin = s.begin; it.count = s.count; it.length = s.length;
    return s.count > 0 && s.count <= p.max_rows_tokens;
}
// Key steps of all row tiles of one head of sequence it.b.
template <int STEP, int KEYS>
__device__ __forceinline__ int64_t decode_head_steps(const DecodeParams& p, DecodeItem it) {
    int64_t n = 0;
    const int tiles = decode_tiles(p, it.count);
    for (it.tile = 0; it.tile < tiles; it.tile += p.head_tiles) {
        decode_range<STEP, KEYS>(p, it);
        n += (int64_t)it.steps * p.head_tiles;
    }
    return n;
}
// The next item of the axis; false at its end.
template <int STEP, int KEYS>
__device__ __forceinline__ bool decode_next(const DecodeParams& p, DecodeItem& it) {
    if (++it.tile >= decode_tiles(p, it.count)) {
        it.tile = 0;
        if (++it.kv_head >= p.c.kv_heads) {
            it.kv_head = 0;
            int b = it.b + 1;
            while (b < p.c.sequences && !decode_sequence(p, b, it)) ++b;
            if (b >= p.c.sequences) return false;
        }
    }
    decode_range<STEP, KEYS>(p, it);
    return true;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
// Two bytes in the low halves of x's 16-bit lanes -> fp16 pair.
__device__ __forceinline__ uint32_t s8_pair(uint32_t x) {
    uint32_t r;                                                   // (x & 0x00ff00ff) ^ 0x64806480 = 1024 + 128 + value
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;\n\tsub.rn.f16x2 %0, %0, %3;" : "=&r"(r) : "r"(x), "r"(0x00ff00ffu), "r"(0x64806480u));
    return r;
}
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t x) {       // the low 16 bits
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(x));
    return r;
}
// One word of a key row (4 dimensions) -> the two A registers of its half of a k16 step.
template <int FORMAT> __device__ __forceinline__ void key_word(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if (FORMAT == RNS_KV_INT8) { lo = s8_pair(w); hi = s8_pair(w >> 8); }
    else { lo = e4m3_pair(w); hi = e4m3_pair(w >> 16); }
}
// Words of the same 4 dimensions of two neighbouring keys -> pairs (key a, key b) of each dimension.
template <int FORMAT> __device__ __forceinline__ void value_words(uint32_t a, uint32_t b, uint32_t (&r)[4]) {
    if (FORMAT == RNS_KV_INT8) {
        r[0] = s8_pair(__byte_perm(a, b, 0x0400)); r[1] = s8_pair(__byte_perm(a, b, 0x0501));
        r[2] = s8_pair(__byte_perm(a, b, 0x0602)); r[3] = s8_pair(__byte_perm(a, b, 0x0703));
    } else {
        const uint32_t lo = __byte_perm(a, b, 0x5140), hi = __byte_perm(a, b, 0x7362);
        r[0] = e4m3_pair(lo); r[1] = e4m3_pair(lo >> 16); r[2] = e4m3_pair(hi); r[3] = e4m3_pair(hi >> 16);
    }
}

template <int DIM, int NT> struct DecodeShape {
    static constexpr int kRows = 8 * NT;
    static constexpr int kKeys = DIM == 256 ? 16 : 32;             // keys of a warp's stage
    static constexpr int kStep = kKeys * kDecodeWarps;
    static constexpr int kHalf = kKeys * DIM;                      // bytes of one side of a stage
    // CTAs of an SM: three where the accumulators leave registers for it (64 sequences up to 8k: 149 us, 173 with
    // two; four, with half the keys a stage, 177)
    static constexpr int kCtas = DIM * NT <= 128 ? 3 : 2;
    static constexpr int kStages = kCtas == 3 ? (DIM == 64 ? 4 : 2) : DIM == 64 ? (NT == 4 ? 5 : 6) : (NT >= 3 || DIM * NT > 256) ? 2 : 3;
    static constexpr int kRing = kDecodeWarps * kStages * 2 * kHalf;
    static constexpr int kStride = DIM + 4;                        // floats between rows of the merge buffer
    static constexpr int kQ = kRows * (DIM + 8) * 2;               // fp16 rows of the tile
    static constexpr int kMerge = kRows * kStride * 4;
    static constexpr int kSmem = 1024 + kRing + kQ + kMerge + kDecodeWarps * kRows * 8 + kRows * 8 +
                                 kDecodeWarps * kStages * (16 + 8) + 64;
    static constexpr int kPartial = kRows * (DIM + 2);             // floats
};

template <int DIM, int NT, int FORMAT>
__global__ void __launch_bounds__(kDecodeThreads, DecodeShape<DIM, NT>::kCtas)
kv_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                 const __grid_constant__ DecodeParams p, int box_rows) {
    using S = DecodeShape<DIM, NT>;
    constexpr int KEYS = S::kKeys, STEP = S::kStep, ROWS = S::kRows, STAGES = S::kStages;
    constexpr int KSTEPS = DIM / 16;                               // k16 steps of the first product
    constexpr int MT = DIM / 16;                                   // m16 tiles of the second
    constexpr bool QREG = KSTEPS * NT <= 16;                       // Q fragments stay in registers
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __half* q_rows = reinterpret_cast<__half*>(smem + S::kRing);
    float* merge = reinterpret_cast<float*>(smem + S::kRing + S::kQ);
    float* warp_m = merge + ROWS * S::kStride;                     // [warps][rows]
    float* warp_l = warp_m + kDecodeWarps * ROWS;
    float* row_scale = warp_l + kDecodeWarps * ROWS;               // [rows] softmax scale / the row's power of two
    float* row_total = row_scale + ROWS;                           // [rows]
    float* scales = row_total + ROWS;                              // [warps][stages][4]: K, K, V, V of the two halves
    const uint32_t bars = smem_addr(scales + kDecodeWarps * STAGES * 4);
    __shared__ int64_t scan[kDecodeWarps];
    __shared__ DecodeItem first_item;
    __shared__ int64_t first_rest;
    __shared__ int abort_word;

    const int t = threadIdx.x, warp = t >> 5, lane = t & 31, r = lane >> 2, c4 = lane & 3;
    const uint32_t ring = smem_addr(smem) + warp * STAGES * 2 * S::kHalf;
    const uint32_t my_bars = bars + warp * STAGES * 8;
    float* my_scales = scales + warp * STAGES * 4;
    if (lane == 0)
        for (int s = 0; s < STAGES; ++s) mbar_init(my_bars + s * 8, 5);
    if (t == 0) abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");

    // --- this CTA's share of the axis of key steps
    const int per = (p.c.sequences + kDecodeThreads - 1) / kDecodeThreads;
    const int b0 = min(t * per, p.c.sequences), b1 = min(b0 + per, p.c.sequences);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) {
        DecodeItem it;
        if (decode_sequence(p, b, it)) mine += decode_head_steps<STEP, KEYS>(p, it) * p.c.kv_heads;
    }
    int64_t upto = mine;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, upto, x);
        if (lane >= x) upto += v;
    }
    if (lane == 31) scan[warp] = upto;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < kDecodeWarps; ++w) {
        if (w < warp) upto += scan[w];
        total += scan[w];
    }
    // neighbours in the axis are neighbours in the grid: no CTA between two of them is without steps
    const int64_t ctas = min((int64_t)gridDim.x, total);
    const int64_t w0 = blockIdx.x < ctas ? total * blockIdx.x / ctas : total;
    const int64_t w1 = blockIdx.x < ctas ? total * (blockIdx.x + 1) / ctas : total;
    if (w0 < w1 && w0 >= upto - mine && w0 < upto) {               // exactly one thread
        int64_t rest = w0 - (upto - mine);
        DecodeItem it;
        for (int b = b0; b < b1; ++b) {
            if (!decode_sequence(p, b, it)) continue;
            const int64_t per_head = decode_head_steps<STEP, KEYS>(p, it);
            if (rest >= per_head * p.c.kv_heads) { rest -= per_head * p.c.kv_heads; continue; }
            it.kv_head = (int)(rest / per_head);
            rest -= it.kv_head * per_head;
            for (it.tile = 0;; ++it.tile) {
                decode_range<STEP, KEYS>(p, it);
                if (rest < it.steps) break;
                rest -= it.steps;
            }
            break;
        }
        first_item = it;
        first_rest = rest;
    }
    __syncthreads();
    int32_t* meta = p.meta + (int64_t)blockIdx.x * 8;
    if (w0 >= w1) {
        if (t == 0) meta[0] = 0;
        return;
    }

    // --- copies: the issuing cursor runs STAGES steps ahead of the consuming one
    DecodeItem ahead = first_item;
    int64_t ahead_left = w1 - w0;
    int ahead_step = (int)first_rest, ahead_slot = 0;
    uint32_t flying = 0;                                           // bit s: slot s was issued and not waited for
    // The page table's entry for the next copy is read one step before it: lanes 0-3, as below.
    int32_t named = -1;
    auto look_up = [&]() {
        const int half_key = ahead.key0 + ahead_step * STEP + warp * KEYS + (KEYS == 32 ? (lane & 1) * 16 : 0);
        if (lane < 4 && ahead_left > 0 && half_key < ahead.length) named = kv_entry(p.c, ahead.b, half_key >> p.c.page_shift);
    };
    look_up();
    auto issue = [&]() {
        if (ahead_left <= 0) return;
        const int key = ahead.key0 + ahead_step * STEP + warp * KEYS;
        if (key < ahead.last && abort_word == 0) {
            flying |= 1u << ahead_slot;
            const uint32_t bar = my_bars + ahead_slot * 8, dst = ring + ahead_slot * 2 * S::kHalf;
            if (lane < 4) {
                // lane = side * 2 + 16-key half: the half's page and its scale of that side
                const int side = lane >> 1, half_key = key + (KEYS == 32 ? (lane & 1) * 16 : 0);
                const int page = half_key < ahead.length ? kv_named(p.c, named) : -1;
                const uint32_t at = smem_addr(my_scales + ahead_slot * 4 + lane);
                if (page >= 0) {
                    const float* src = (side ? p.c.scale[1] : p.c.scale[0]) + (int64_t)page * p.c.kv_heads + ahead.kv_head;
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(at), "l"(src) : "memory");
                } else {
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(0.0f) : "memory");
                }
                if (lane == 0) mbar_arrive_expect_tx(bar, 2 * S::kHalf);
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
                __syncwarp(0xf);
                // a bad page loads from behind the last one: zeros
                const bool boxes = KEYS == 16 || box_rows == 16 || (lane & 1) == 0;
                if (boxes && (KEYS == 32 || (lane & 1) == 0)) {
                    const CUtensorMap* map = side ? &map_v : &map_k;
                    const int row = ahead.kv_head * p.c.page_tokens + (half_key & (p.c.page_tokens - 1));
                    const int z = page >= 0 ? page : (int)p.c.pages;
                    const uint32_t to = dst + side * S::kHalf + (KEYS == 32 ? (lane & 1) * 16 : 0) * (DIM == 64 ? 64 : 128);
                    tma_load_3d(to, map, bar, 0, row, z);
                    if (DIM == 256) tma_load_3d(to + KEYS * 128, map, bar, 128, row, z);
                }
            }
        }
        if (++ahead_slot == STAGES) ahead_slot = 0;
        if (--ahead_left > 0 && ++ahead_step == ahead.steps) {
            ahead_step = 0;
            decode_next<STEP, KEYS>(p, ahead);
        }
        look_up();
    };
#pragma unroll 1
    for (int s = 0; s < STAGES; ++s) issue();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the joining kernel may take its place and wait

    // --- items
    DecodeItem it = first_item;
    int step = (int)first_rest, slot = 0;
    uint32_t parity = 0;                                           // bit s: phase of slot s
    int64_t left = w1 - w0;
    bool alive = true, begins = step == 0;
    if (t == 0) meta[0] = 0;
    for (;;) {
        const int steps_here = (int)min((int64_t)(it.steps - step), left);
        const int tile_t0 = it.tile / p.head_tiles * p.token_tile, tile_h0 = it.tile % p.head_tiles * p.head_tile;
        const int n_tokens = min(p.token_tile, it.count - tile_t0), n_heads = min(p.head_tile, p.a.group - tile_h0);
        const int head0 = it.kv_head * p.a.group + tile_h0;
        // queries of the tile as fp16, each row times a power of two that brings its largest element to [2^7, 2^8)
        // (all of a warp's rows are fetched before the first is looked at: it is their latency that counts)
        constexpr int MINE = ROWS / kDecodeWarps, PER = DIM / 32;
        float v[MINE][PER];
#pragma unroll
        for (int n = 0; n < MINE; ++n) {
            const int row = warp + n * kDecodeWarps, tok = row / p.head_tile, hd = row - tok * p.head_tile;
            const bool there = tok < n_tokens && hd < n_heads;
            const int64_t at = (it.begin + tile_t0 + tok) * p.a.q_token_stride + (int64_t)(head0 + hd) * p.a.q_head_stride + lane;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                v[n][i] = 0.0f;
                if (there && lane + i * 32 < p.c.head_dim)
                    v[n][i] = p.a.type == RNS_F16 ? __half2float(static_cast<const __half*>(p.a.q)[at + i * 32])
                                                  : __bfloat162float(static_cast<const __nv_bfloat16*>(p.a.q)[at + i * 32]);
            }
        }
#pragma unroll
        for (int n = 0; n < MINE; ++n) {
            const int row = warp + n * kDecodeWarps;
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < PER; ++i) top = fmaxf(top, fabsf(v[n][i]));
            const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
            const int e = (int)(bits >> 23);                       // biased exponent of the largest element
            const bool plain = bits == 0 || e == 255;
            // 2^(134 - e): representable for every e of a finite bf16 or fp16 element that is not tiny
            const int shift = plain ? 0 : max(-126, min(120, 134 - e));
            const float up = __uint_as_float((uint32_t)(shift + 127) << 23);
            const float down = __uint_as_float((uint32_t)(127 - max(-120, min(126, shift))) << 23);
#pragma unroll
            for (int i = 0; i < PER; ++i) q_rows[row * (DIM + 8) + lane + i * 32] = __float2half_rn(v[n][i] * up);
            if (lane == 0) row_scale[row] = p.a.scale_log2 * down;
        }
        __syncthreads();
        // fragments: dims d .. d+3 of a thread belong to one word of a key row
        uint32_t qf[QREG ? KSTEPS : 1][NT][2];
        auto load_q = [&](int ks, uint32_t (&f)[NT][2]) {
            const int word = ks & 3, chunk = ks >> 2;              // 16-byte chunk of the thread: see key offsets below
            const int d = (DIM == 64 ? c4 * 16 : (chunk >> 1) * 128 + (2 * c4 + (chunk & 1)) * 16) + word * 4;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const uint2 w = *reinterpret_cast<const uint2*>(q_rows + (nt * 8 + r) * (DIM + 8) + d);
                if (FORMAT == RNS_KV_INT8) {
                    f[nt][0] = __byte_perm(w.x, w.y, 0x5410);      // (d, d+2)
                    f[nt][1] = __byte_perm(w.x, w.y, 0x7632);      // (d+1, d+3)
                } else { f[nt][0] = w.x; f[nt][1] = w.y; }
            }
        };
        if (QREG) {
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ++ks) load_q(ks, qf[QREG ? ks : 0]);
        }
        float q_scale[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            q_scale[nt][0] = row_scale[nt * 8 + 2 * c4];
            q_scale[nt][1] = row_scale[nt * 8 + 2 * c4 + 1];
        }
        // keys every row of the tile sees
        const int position = it.length - it.count + tile_t0;
        const int all_last = p.a.causal ? position + 1 : position >= 0 ? it.length : 0;
        const int all_first = kv_first_key(p.a, position + n_tokens - 1);
        const int tile_first = kv_first_key(p.a, position);

        // and those that each of this thread's rows sees: [sees0, sees1)
        int sees0[NT][2], sees1[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int pos = position + (nt * 8 + 2 * c4 + e) / p.head_tile;
                sees1[nt][e] = pos < 0 ? 0 : p.a.causal ? pos + 1 : it.length;
                sees0[nt][e] = kv_first_key(p.a, pos);
            }

        float o[MT][NT][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][nt][e] = 0.0f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) { m[nt][0] = m[nt][1] = kNoMax; l[nt][0] = l[nt][1] = 0.0f; }

        for (int n = 0; n < steps_here; ++n, ++step) {
            const int key = it.key0 + step * STEP + warp * KEYS;
            if (key < it.last) {
                if (alive) alive = warp_wait_bounded(my_bars + slot * 8, (parity >> slot) & 1, &abort_word, wait_code(1, slot));
                if (alive) { parity ^= 1u << slot; flying &= ~(1u << slot); }
                const uint32_t k_base = ring + slot * 2 * S::kHalf, v_base = k_base + S::kHalf;
                if (alive) {
#pragma unroll 1
                    for (int half = 0; half < KEYS / 16; ++half) {
                        const int k0 = key + half * 16;
                        if (k0 >= it.last) break;
                        if (k0 + 16 <= tile_first) continue;
                        const float k_scale = my_scales[slot * 4 + half];
                        const KvValueScale vs = kv_value_scale(my_scales[slot * 4 + 2 + half]);
                        // two chains of products for each tile, so that they do not wait for one another
                        float s[NT][4], s2[NT][4];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[nt][e] = s2[nt][e] = 0.0f;
#pragma unroll
                        for (int chunk = 0; chunk < DIM / 64; ++chunk) {
                            // rows r and r + 8; a thread's chunks are 16 bytes, swizzled by the copy
                            uint32_t at;
                            if (DIM == 64) at = k_base + (half * 16 + r) * 64 + ((c4 ^ ((r >> 1) & 3)) << 4);
                            else at = k_base + (chunk >> 1) * KEYS * 128 + (half * 16 + r) * 128 + (((2 * c4 + (chunk & 1)) ^ r) << 4);
                            const uint4 x = lds128(at), y = lds128(at + (DIM == 64 ? 512 : 1024));
                            const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                            for (int w = 0; w < 4; ++w) {
                                uint32_t a0, a1, a2, a3;
                                key_word<FORMAT>(xw[w], a0, a2);
                                key_word<FORMAT>(yw[w], a1, a3);
                                uint32_t f[NT][2];
                                if (!QREG) load_q(chunk * 4 + w, f);
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt)
                                    mma_f16(NT < 3 && (w & 1) ? s2[nt] : s[nt], a0, a1, a2, a3, QREG ? qf[QREG ? chunk * 4 + w : 0][nt][0] : f[nt][0],
                                            QREG ? qf[QREG ? chunk * 4 + w : 0][nt][1] : f[nt][1]);
                            }
                        }
                        const bool whole = k0 + 16 <= all_last && k0 >= all_first;
                        bool grow = false;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[nt][e] = (s[nt][e] + s2[nt][e]) * (q_scale[nt][e & 1] * k_scale);
                        }
                        if (!whole) {
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const int j = k0 + r + (e >> 1) * 8;
                                    if (j < sees0[nt][e & 1] || j >= sees1[nt][e & 1]) s[nt][e] = -INFINITY;
                                }
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) grow = grow || s[nt][e] > m[nt][e & 1] - vs.exponent + kLag;
                        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    float top = fmaxf(s[nt][e], s[nt][e + 2]);
#pragma unroll
                                    for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                                    top = top > m[nt][e] - vs.exponent + kLag ? ceilf(top + vs.exponent) : m[nt][e];  // a row's result is its own affair
                                    const float keep = exp2_approx(m[nt][e] - top);
                                    m[nt][e] = top;
                                    l[nt][e] *= keep;
#pragma unroll
                                    for (int i = 0; i < MT; ++i) { o[i][nt][e] *= keep; o[i][nt][e + 2] *= keep; }
                                }
                        }
                        uint32_t pf[NT][2], pl[NT][2];                             // weights, and what rounding left of them
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            float w[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float pe = exp2_approx(s[nt][e] - (m[nt][e & 1] - vs.exponent));
                                l[nt][e & 1] = fmaf(pe, vs.back, l[nt][e & 1]);
                                w[e] = pe * vs.weight;
                                if (!whole && s[nt][e] == -INFINITY) w[e] = 0.0f;      // not NaN from the page's scale
                            }
                            const __half2 top = __floats2half2_rn(w[0], w[1]), low = __floats2half2_rn(w[2], w[3]);
                            pf[nt][0] = transpose8x8(*reinterpret_cast<const uint32_t*>(&top));
                            pf[nt][1] = transpose8x8(*reinterpret_cast<const uint32_t*>(&low));
                            const float2 t2 = __half22float2(top), l2 = __half22float2(low);
                            const __half2 top_left = __floats2half2_rn(w[0] - t2.x, w[1] - t2.y);
                            const __half2 low_left = __floats2half2_rn(w[2] - l2.x, w[3] - l2.y);
                            pl[nt][0] = transpose8x8(*reinterpret_cast<const uint32_t*>(&top_left));
                            pl[nt][1] = transpose8x8(*reinterpret_cast<const uint32_t*>(&low_left));
                        }
                        // values: keys 2c, 2c+1, 2c+8, 2c+9; 16 (DIM 64: 8) dimensions of this thread
                        const bool tail = FORMAT == RNS_KV_E4M3 && k0 + 16 > it.length;
#pragma unroll
                        for (int part = 0; part < (DIM == 256 ? 2 : 1); ++part) {
                            constexpr int WORDS = DIM == 64 ? 2 : 4;
                            uint32_t x[4][WORDS];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int row = 2 * c4 + (i & 1) + (i >> 1) * 8;
                                if (DIM == 64) {
                                    const uint2 v = lds64(v_base + (half * 16 + row) * 64 + (((r >> 1) ^ ((row >> 1) & 3)) << 4) + (r & 1) * 8);
                                    x[i][0] = v.x; x[i][1] = v.y;
                                } else {
                                    const uint4 v = lds128(v_base + part * KEYS * 128 + (half * 16 + row) * 128 + ((r ^ (row & 7)) << 4));
                                    x[i][0] = v.x; x[i][1] = v.y; x[i][WORDS - 2] = v.z; x[i][WORDS - 1] = v.w;
                                }
                                // bytes behind the sequence may be NaN patterns, which no weight of zero removes
                                if (tail && k0 + row >= it.length) {
#pragma unroll
                                    for (int w = 0; w < WORDS; ++w) x[i][w] = 0;
                                }
                            }
#pragma unroll
                            for (int w = 0; w < WORDS; ++w) {
                                uint32_t a[4], b[4];
                                value_words<FORMAT>(x[0][w], x[1][w], a);
                                value_words<FORMAT>(x[2][w], x[3][w], b);
#pragma unroll
                                for (int h = 0; h < 2; ++h)
#pragma unroll
                                    for (int nt = 0; nt < NT; ++nt)
                                        mma_f16(o[part * 8 + w * 2 + h][nt], a[2 * h], a[2 * h + 1], b[2 * h], b[2 * h + 1], pf[nt][0], pf[nt][1]);
#pragma unroll
                                for (int h = 0; h < 2; ++h)
#pragma unroll
                                    for (int nt = 0; nt < NT; ++nt)
                                        mma_f16(o[part * 8 + w * 2 + h][nt], a[2 * h], a[2 * h + 1], b[2 * h], b[2 * h + 1], pl[nt][0], pl[nt][1]);
                            }
                        }
                    }
                    __syncwarp();                                  // the slot is read: it may be filled again
                }
            }
            issue();
            if (++slot == STAGES) slot = 0;
        }
        left -= steps_here;
        const bool ends = step == it.steps;

        // --- the four warps' parts meet
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], x);
                if (r == 0) {
                    warp_m[warp * ROWS + nt * 8 + 2 * c4 + e] = m[nt][e];
                    warp_l[warp * ROWS + nt * 8 + 2 * c4 + e] = l[nt][e];
                }
            }
        __syncthreads();
        float factor[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float top = kNoMax;
#pragma unroll
                for (int w = 0; w < kDecodeWarps; ++w) top = fmaxf(top, warp_m[w * ROWS + nt * 8 + 2 * c4 + e]);
                factor[nt][e] = exp2_approx(m[nt][e] - top);
            }
#pragma unroll 1
        for (int w = 0; w < kDecodeWarps; ++w) {
            if (warp == w) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int d = DIM == 64 ? r * 8 + 2 * i : (i >> 3) * 128 + r * 16 + 2 * (i & 7);
                            float2* at = reinterpret_cast<float2*>(merge + (nt * 8 + 2 * c4 + e) * S::kStride + d);
                            float2 v = make_float2(o[i][nt][e] * factor[nt][e], o[i][nt][e + 2] * factor[nt][e]);
                            if (w > 0) { v.x += at->x; v.y += at->y; }
                            *at = v;
                        }
            }
            __syncthreads();
        }
        if (t < ROWS) {
            float top = kNoMax, sum = 0.0f;
            for (int w = 0; w < kDecodeWarps; ++w) top = fmaxf(top, warp_m[w * ROWS + t]);
            for (int w = 0; w < kDecodeWarps; ++w) sum += warp_l[w * ROWS + t] * exp2_approx(warp_m[w * ROWS + t] - top);
            row_scale[t] = top;
            row_total[t] = sum;
        }
        __syncthreads();
        if (begins && ends) {
            for (int row = warp; row < ROWS; row += kDecodeWarps) {
                const int tok = row / p.head_tile, hd = row - tok * p.head_tile;
                if (tok >= n_tokens || hd >= n_heads) continue;
                const int64_t token = it.begin + tile_t0 + tok, head = head0 + hd;
                const float sum = row_total[row], inv = row_scale[row] == kNoMax && sum == 0.0f ? 0.0f : 1.0f / sum;
                for (int d = lane; d < p.c.head_dim; d += 32) {
                    const float v = merge[row * S::kStride + d] * inv;
                    const int64_t at = token * p.a.out_token_stride + head * p.a.out_head_stride + d;
                    if (p.a.type == RNS_F16) static_cast<__half*>(p.a.out)[at] = __float2half_rn(v);
                    else static_cast<__nv_bfloat16*>(p.a.out)[at] = __float2bfloat16_rn(v);
                }
                if (p.a.lse != nullptr && lane == 0)
                    p.a.lse[token * p.a.heads + head] = inv == 0.0f ? -INFINITY : (row_scale[row] + log2f(sum)) * 0.6931471805599453f;
            }
        } else {
            float* part = p.partial + ((int64_t)blockIdx.x * 2 + (left + steps_here == w1 - w0 ? 0 : 1)) * S::kPartial;
            if (t < ROWS) { part[t] = row_scale[t]; part[ROWS + t] = row_total[t]; }
            for (int i = t; i < ROWS * DIM; i += kDecodeThreads) part[2 * ROWS + i] = merge[i / DIM * S::kStride + i % DIM];
            if (begins && t == 0) {
                // this CTA holds the first piece: it names the item and where its pieces are
                const int64_t end = w1 - left - steps_here + it.steps;      // of the item, on the axis
                int64_t lastcta = (end - 1) * ctas / total;
                while (total * (lastcta + 1) / ctas < end) ++lastcta;
                while (total * lastcta / ctas > end - 1) --lastcta;
                meta[1] = (int)(lastcta - blockIdx.x) + 1;
                meta[2] = left + steps_here == w1 - w0 ? 0 : 1;
                meta[3] = it.b; meta[4] = it.kv_head; meta[5] = it.tile;
                meta[0] = 1;
            }
        }
        if (left <= 0) break;
        step = 0;
        begins = true;
        decode_next<STEP, KEYS>(p, it);
        __syncthreads();                                           // the buffers above are free again
    }
    // after an expired wait: copies still in flight get another bounded while to land
    for (int s = 0; flying != 0 && s < STAGES; ++s)
        for (int i = 0; ((flying >> s) & 1) && i < 10000 && !mbar_try_wait(my_bars + s * 8, (parity >> s) & 1); ++i) {}
    if (abort_word != 0 && t == 0 && p.c.status != nullptr) *p.c.status = RNS_ERR_DEVICE_TIMEOUT;
}

// Joins the pieces of the items that a CTA boundary cut: block (first piece's CTA, row).
template <int DIM, int NT>
__global__ void __launch_bounds__(128) kv_join_kernel(const __grid_constant__ DecodeParams p) {
    using S = DecodeShape<DIM, NT>;
    asm volatile("griddepcontrol.wait;" ::: "memory");             // the pieces are complete and visible
    const int32_t* meta = p.meta + (int64_t)blockIdx.x * 8;
    if (meta[0] == 0) return;
    const int row = blockIdx.y, pieces = meta[1], slot = meta[2], kv_head = meta[4], tile = meta[5];
    const KvSpan s = kv_span(p.c, p.a.lens, p.a.starts, p.a.tokens, meta[3]);
    const int tok = tile / p.head_tiles * p.token_tile + row / p.head_tile, hd = tile % p.head_tiles * p.head_tile + row % p.head_tile;
    if (tok >= s.count || hd >= p.a.group || row >= p.token_tile * p.head_tile) return;
    // piece 0 lies in this CTA's slot, piece i in slot 0 of the i-th CTA after it
    const float* first = p.partial + ((int64_t)blockIdx.x * 2 + slot) * S::kPartial;
    const float* next = p.partial + (int64_t)blockIdx.x * 2 * S::kPartial;
    const auto piece = [&](int i) { return i == 0 ? first : next + (int64_t)i * 2 * S::kPartial; };
    __shared__ float factors[128], tops[4];
    const int t = threadIdx.x;
    float top = kNoMax;
    for (int i = t; i < pieces; i += 128) top = fmaxf(top, piece(i)[row]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    if ((t & 31) == 0) tops[t >> 5] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    float sum = 0.0f, o[DIM > 128 ? 2 : 1] = {};
    for (int base = 0; base < pieces; base += 128) {               // pieces in key order, their loads in flight together
        const int n = min(128, pieces - base);
        __syncthreads();
        if (t < n) factors[t] = exp2_approx(piece(base + t)[row] - top);
        __syncthreads();
#pragma unroll 8
        for (int i = 0; i < n; ++i) {
            const float* part = piece(base + i);
            const float f = factors[i];
            sum = fmaf(part[S::kRows + row], f, sum);
#pragma unroll
            for (int j = 0; j < (DIM > 128 ? 2 : 1); ++j) {
                const int d = min(t + j * 128, DIM - 1);
                o[j] = fmaf(part[2 * S::kRows + row * DIM + d], f, o[j]);
            }
        }
    }
    const float inv = top == kNoMax && sum == 0.0f ? 0.0f : 1.0f / sum;
    const int64_t token = s.begin + tok, head = (int64_t)kv_head * p.a.group + hd;
#pragma unroll
    for (int j = 0; j < (DIM > 128 ? 2 : 1); ++j) {
        const int d = threadIdx.x + j * 128;
        if (d >= p.c.head_dim) continue;
        const int64_t at = token * p.a.out_token_stride + head * p.a.out_head_stride + d;
        if (p.a.type == RNS_F16) static_cast<__half*>(p.a.out)[at] = __float2half_rn(o[j] * inv);
        else static_cast<__nv_bfloat16*>(p.a.out)[at] = __float2bfloat16_rn(o[j] * inv);
    }
    if (p.a.lse != nullptr && threadIdx.x == 0)
        p.a.lse[token * p.a.heads + head] = inv == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int sm_count(int* out) {
    static std::atomic<int> known[64];                             // per device, looked up once
    int dev = 0;
    RNS_CUDA_OK(cudaGetDevice(&dev));
    int n = dev < 64 ? known[dev].load(std::memory_order_relaxed) : 0;
    if (n == 0) {
        RNS_CUDA_OK(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
        if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
    }
    *out = n;
    return RNS_OK;
}
int allow_smem(const void* kernel, int bytes, std::atomic<uint64_t>* done) {
    int dev = 0;
    RNS_CUDA_OK(cudaGetDevice(&dev));
    if (dev < 64 && (done->load(std::memory_order_relaxed) >> dev & 1)) return RNS_OK;
    RNS_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (dev < 64) done->fetch_or(1ull << dev, std::memory_order_relaxed);
    return RNS_OK;
}

// Rows of a tile in eights: the smallest that holds the rows of one head and sequence, up to 32
// (16 for heads above 128, whose accumulators fill the registers).  Each eight costs its products, its
// exponentials and 4 * head_dim / 16 registers: 20 rows (5 tokens x 4 heads of 80, 16 sequences) take
// 36.7 us in a tile of 24 and 42.6 us in one of 32.
static int decode_nt(const KvView& c, const KvQuery& a, int max_new) {
    const int64_t rows = (int64_t)max_new * a.group;
    if (rows <= 8) return 1;
    if (rows <= 16 || c.head_dim > 128) return 2;
    if (rows <= 24) return 3;
    return 4;
}
static int decode_dim(const KvView& c) { return c.head_dim <= 64 ? 64 : c.head_dim <= 128 ? 128 : 256; }

int64_t kv_decode_workspace(const KvView& c, const KvQuery& a, int max_new) {
    int sms = 0;
    if (sm_count(&sms) != RNS_OK) return -RNS_ERR_CUDA;
    const int64_t rows = 8 * decode_nt(c, a, max_new);
    return (int64_t)kDecodeMostCtas * sms * (2 * rows * (decode_dim(c) + 2) * 4 + 32);
}

template <int DIM, int NT, int FORMAT>
static int launch_decode(DecodeParams& p, void* workspace, cudaStream_t st) {
    using S = DecodeShape<DIM, NT>;
    static_assert(S::kCtas * (S::kSmem + 1024 + 256) <= 228 * 1024, "shared memory of an SM");
    int sms = 0;
    if (int rc = sm_count(&sms)) return rc;
    CUtensorMap maps[2];
    const int box_rows = min(S::kKeys, p.c.page_tokens);
    for (int i = 0; i < 2; ++i) {
        const uint64_t dims[3] = {(uint64_t)p.c.head_dim, (uint64_t)p.c.kv_heads * p.c.page_tokens, (uint64_t)p.c.pages};
        const uint64_t strides[2] = {dims[0], dims[0] * dims[1]};
        const uint32_t box[3] = {DIM == 64 ? 64u : 128u, (uint32_t)box_rows, 1u};
        if (int rc = make_map(&maps[i], p.c.data[i], 3, dims, strides, box, DIM == 64 ? 64 : 128)) return rc;
    }
    const int grid = S::kCtas * sms;
    p.meta = static_cast<int32_t*>(workspace);
    p.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + (int64_t)grid * 32);
    const int rows = S::kRows;
    p.head_tile = min(p.a.group, rows);
    p.token_tile = rows / p.head_tile;
    p.head_tiles = (p.a.group + p.head_tile - 1) / p.head_tile;
    const auto kernel = kv_decode_kernel<DIM, NT, FORMAT>;
    static std::atomic<uint64_t> allowed{0};
    if (int rc = allow_smem(reinterpret_cast<const void*>(kernel), S::kSmem, &allowed)) return rc;
    kernel<<<grid, kDecodeThreads, S::kSmem, st>>>(maps[0], maps[1], p, box_rows);
    RNS_CUDA_OK(cudaGetLastError());
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid, (unsigned)(p.token_tile * p.head_tile));
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    RNS_CUDA_OK(cudaLaunchKernelEx(&cfg, kv_join_kernel<DIM, NT>, p));
    return RNS_OK;
}

int kv_decode(const KvView& c, const KvQuery& a, int format, int max_new, int max_rows_tokens, void* workspace, cudaStream_t st) {
    DecodeParams p;
    memset(&p, 0, sizeof(p));
    p.c = c; p.a = a;
    p.max_rows_tokens = max_rows_tokens;
    const int dim = decode_dim(c), nt = decode_nt(c, a, max_new);
#define RNS_KV_DECODE(D, N)                                                                        \
    if (dim == D && nt == N)                                                                       \
        return format == RNS_KV_INT8 ? launch_decode<D, N, RNS_KV_INT8>(p, workspace, st)          \
                                     : launch_decode<D, N, RNS_KV_E4M3>(p, workspace, st)
    RNS_KV_DECODE(64, 1);
    RNS_KV_DECODE(64, 2);
    RNS_KV_DECODE(64, 3);
    RNS_KV_DECODE(64, 4);
    RNS_KV_DECODE(128, 1);
    RNS_KV_DECODE(128, 2);
    RNS_KV_DECODE(128, 3);
    RNS_KV_DECODE(128, 4);
    RNS_KV_DECODE(256, 1);
    RNS_KV_DECODE(256, 2);
#undef RNS_KV_DECODE
    return fail(RNS_ERR_UNSUPPORTED, "no decode kernel for this head size");
}

}  // namespace rns

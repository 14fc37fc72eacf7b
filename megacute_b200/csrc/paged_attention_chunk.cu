// Attention over a paged cache for items of up to 256 rows (new tokens x heads of a group): chunks of prompts, whole prompts, batches that
// mix them with single tokens.
//
// An item is two tiles of 128 query rows that share every tile of 128 keys (paged_attention.cuh: a unit).  One block per SM, one worker per block:
//   warps 0-3, 4-7   softmax of tile 0 and 1, one thread per row (a lane of tensor memory), so that nothing is exchanged between threads: the
//                    row's 128 scores are read twice, 64 columns at a time, for the maximum and for the weights; log2 domain, scale * log2(e)
//                    folded into the subtraction; the maximum is only raised when it grows by more than 2^8, and then the row of O in tensor
//                    memory is scaled down; results
//   warp 8           loader: walks the block's items and tells the other roles; Q as boxes of 64 columns x group heads x tokens, K and V as boxes of 64 columns x the rows of a page (at most 128), found
//                    through the page table, into one ring of tiles in the order K, V, K, V, ...
//   warp 9           products: S = Q K^T and O += P V on tcgen05, S, P (over S) and O in tensor memory
//   warps 10, 11     look at every V tile before it is multiplied: rows that no token of the item sees become zeros (they may hold anything, and
//                    0 * inf is no number); where some tokens see a row and others do not, values that are no numbers are taken out and added back
//                    to the rows that see them when the item ends
// P is rounded to the operand type, which the second product takes; sums of weights are of the unrounded ones, O and both statistics fp32.
//
// What bounds it: a score product of 128 x 128 x 64 and its P V take 256 cycles each of the tensor cores, the 16384 exponentials 1024 of the special
// function units (16 a cycle) or 768 with a quarter of them on the fp32 units, and the maxima, conversions and accesses to tensor memory of the same
// threads come on top.  So head_dim 64 is bound by the softmax; for 128, whose products take twice as long, the chain from S over P to P V and the next S
// through two buffers of scores counts as much.  Measured as captured graphs: 4 prompts of 4096 tokens, bf16, 32 heads and 8 kv heads of 64: 386 to 394 us,
// 697 to 712 TFLOP/s (called one by one 409 to 420 us); 16 heads and 4 kv heads of 128: 271 us, 1014 TFLOP/s; 509 tokens behind 16001, 32 heads of 64: 100 us,
// 675 TFLOP/s (104).
// Both sides of the choices, for the first two of these when they took 400 and 283 us: the maximum raised whenever it grows 459 and 333; the row's scores held in registers
// (spills) 467; two threads a row 429; the two tiles' exponentials in turns 458.
// Every wait has a limit, after which the block counts it, raises a flag that all its waits ask for, waits for its copies, frees its tensor memory and
// ends; mk_paged_attention_failures tells the count.
#include <cuda.h>          // CUtensorMap

#include "paged_attention.cuh"
#include "tc.cuh"

namespace mk {

__device__ unsigned g_paged_failed;                   // grows when a block gives up waiting; never put back, so that no reader takes it from another

namespace {

constexpr int kChunkThreads = 384;
constexpr float kLazy = 8.0f;                         // (log2; fp32 sums and products of weights up to 2^8 lose nothing, and fp16 weights stay in range)
// Of eight pairs of exponentials, those that the fp32 units take.  4 x 4096 tokens with none, one, two, three, four of them, when two took 400 and 283 us:
// 419, 404, 400, 406, 419 (64-wide heads), 292, 287, 283, 279, 284 (128-wide; since then 271, 270, 282 with two, three, four).
constexpr uint32_t kFmaPairs = 0b00010001;
template <bool V> struct Const { static constexpr bool value = V; };
constexpr unsigned long long kWaitNs = 2000000000ull;
constexpr int kTileRows = 128;
constexpr int kSubBytes = kTileRows * 128;            // 64 columns of a tile of 128 rows
constexpr int kSeen = 32;                             // entries of the ring of tile descriptions, far more than tiles in flight
constexpr int kRingBars = 8;                          // barriers of key tiles, more than tiles in the ring
constexpr int kOddTiles = 6;                          // tiles of an item that some tokens see in part: at most three at either end

template <int D> struct Map {
    static constexpr int kSubs = D / 64;
    static constexpr int kTile = kSubs * kSubBytes;
    static constexpr int kSlots = D == 64 ? 10 : 5;   // tiles in the ring
    static constexpr int kQ = 0, kRing = 2 * kTile, kBytes = kRing + kSlots * kTile;       // (Sync lies behind)
    static constexpr int kScores = D == 64 ? 3 : 2;   // tensor-memory buffers of scores, 128 columns each from column 0
    static constexpr uint32_t kO = kScores * 128;     // ... then O of tile 0 and of tile 1
};

// What the block does to one item.  The loader finds it and tells the other roles through a short ring in shared memory.
struct Part {
    int tokens, row0, block, s;                       // its tokens, first row of the packed batch, block of heads, sequence
    int lo, hi;                                       // keys some token sees
    int first_lo, first_hi;                           // keys the first token sees, the next one's are one further (saturated far outside of what there is)
    int key0, units, tiles;                           // first key of the part; key tiles (0: no more items); query tiles
    int whole;                                        // bit 0: it begins the item, bit 1: it ends it
};
constexpr int kShift = 7;
constexpr int kParts = 4;                             // entries of that ring
__device__ __forceinline__ int saturated(long long x) { return (int)min(max(x, -0x7fff0000ll), 0x7fffff00ll); }
__device__ __forceinline__ Part part_of(const AttnArgs& a, const Walk<kShift>& w) {
    Part p;
    p.tokens = w.item_tokens(a);
    p.row0 = w.r0 + w.t;
    p.block = w.kv;
    p.s = w.s;
    p.lo = w.item.lo;
    p.hi = w.item.hi;
    p.first_hi = saturated(w.p + w.t);
    p.first_lo = a.window > 0 ? saturated(w.p + w.t + 1 - a.window) : -0x7fff0000;
    p.key0 = w.item.key0 + (w.unit << kShift);
    p.units = w.stop - w.unit;
    p.tiles = p.tokens > a.tokens / 2 ? 2 : 1;
    p.whole = (w.unit == 0 ? 1 : 0) | (w.stop == w.item.units ? 2 : 0);
    return p;
}
// keys that every token of [t0, t1) sees
__device__ __forceinline__ void seen_by_all(const Part& p, int t0, int t1, int& lo, int& hi) {
    hi = min(p.first_hi + t0, p.hi);
    lo = max(p.first_lo + t1 - 1, 0);
}
__device__ __forceinline__ void seen_by(const Part& p, int token, int& lo, int& hi) { seen_by_all(p, token, token + 1, lo, hi); }

struct Sync {
    // (by parity a wait only tells a phase from the one in front of it: a barrier's phases are all waited for by the same threads, one after the
    // other, or the one in front is known to be over)
    unsigned long long q_full, q_free;                // one per item
    unsigned long long k_full[kRingBars], v_full[kRingBars], v_ready[kRingBars];           // key tile c: c % kRingBars
    unsigned long long slot_free[10];                 // slots of the ring of tiles
    unsigned long long s_full[2][4], p_full[2][4], pv_done[2][4];                          // tile t's k-th block of scores: k % 4
    unsigned long long o_free[2], part_full[kParts], part_free[kParts];
    uint32_t tmem;
    int abort;
    uint32_t there[kSeen];                            // bit b: keys [16 b, 16 b + 16) of the tile are loaded
    uint32_t odd[kParts][kOddTiles][4];               // keys of the item's n-th partial tile with values that are no numbers
    int odd_any[kParts];
    Part part[kParts];
};

// All lanes of a warp wait for one phase.  Asked once in line; the rest, with the limit, is a call, so that the roles' loops stay short.
__device__ __noinline__ bool wait_longer(Sync* s, uint32_t bar, uint32_t parity) {
    auto* const at = reinterpret_cast<unsigned long long*>(__cvta_shared_to_generic(bar));
    const unsigned long long t0 = globaltimer();
    bool ok;
    // (try_wait suspends the warp: what asks again and again takes issue slots from the softmax)
    while (!(ok = mbar_try_wait(at, parity)) && !*(volatile int*)&s->abort) {
        if (globaltimer() - t0 > kWaitNs) {
            *(volatile int*)&s->abort = 1;
            atomicAdd(&g_paged_failed, 1u);
            break;
        }
    }
    return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ bool warp_wait(Sync* s, unsigned long long* bar, uint32_t parity) {
    if (__all_sync(0xffffffffu, mbar_test_wait(bar, parity))) return true;
    return wait_longer(s, smem_u32(bar), parity);
}
// The next item: all lanes of a warp of a role other than the loader.  False: there is none, or a wait gave up.
__device__ __forceinline__ bool next_part(Sync* s, uint32_t items, Part& p) {
    if (!warp_wait(s, &s->part_full[items % kParts], (items / kParts) & 1u)) return false;
    p = s->part[items % kParts];
    return p.units > 0;
}
// ... and done with it
__device__ __forceinline__ void done_part(Sync* s, uint32_t items) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&s->part_free[items % kParts]);
}
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* m, int x, int y, unsigned long long* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(m),
                 "r"(x), "r"(y), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* m, int x, int y, int z, unsigned long long* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(m),
                 "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t* w) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at),
        "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]), "r"(w[8]), "r"(w[9]), "r"(w[10]),
        "r"(w[11]), "r"(w[12]), "r"(w[13]), "r"(w[14]), "r"(w[15])
        : "memory");
}
// 32 columns of this thread's lane, not waited for
__device__ __forceinline__ void tmem_ld32(uint32_t at, float* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
        "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
          "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]),
          "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]),
          "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void use32(float* v) {                             // what was loaded is read behind this point (the wait in front of it)
#pragma unroll
    for (int e = 0; e < 32; ++e) asm volatile("" : "+f"(v[e]));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D (+)= A B with A in tensor memory
__device__ __forceinline__ void mma_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d), "r"(a), "l"(b),
                 "r"(idesc), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ float2 fma_2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{ .reg .b64 x, y, z, w; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mov.b64 z, {%6, %7}; fma.rn.f32x2 w, x, y, z; mov.b64 {%0, %1}, w; }"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add_2(float2 a, float2 b) {
    float2 d;
    asm("{ .reg .b64 x, y, w; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; add.rn.f32x2 w, x, y; mov.b64 {%0, %1}, w; }"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
// 2^y of a pair without the special function units: y = n + f, n whole, |f| <= 1/2; 2^f by the polynomial of degree 4 whose relative error
// is least over that range (2^-18.5, computed with Remez' exchange), n added to its exponent.  For y in [-inf, 127), as 2^-125 below that; not for NaN.
__device__ __forceinline__ float2 ex2_fma(float2 y) {
    const float2 big = make_float2(12582912.f, 12582912.f);                    // 1.5 * 2^23: the sum's last bit is one
    y = make_float2(fmaxf(y.x, -125.f), fmaxf(y.y, -125.f));
    const float2 t = add_2(y, big), n = add_2(t, make_float2(-big.x, -big.y)), f = fma_2(n, make_float2(-1.f, -1.f), y);
    float2 q = fma_2(f, make_float2(0x1.3997d6p-7f, 0x1.3997d6p-7f), make_float2(0x1.ca1440p-5f, 0x1.ca1440p-5f));
    q = fma_2(q, f, make_float2(0x1.ec06dap-3f, 0x1.ec06dap-3f));
    q = fma_2(q, f, make_float2(0x1.62e0dcp-1f, 0x1.62e0dcp-1f));
    q = fma_2(q, f, make_float2(0x1.ffffe8p-1f, 0x1.ffffe8p-1f));
    return make_float2(__int_as_float(__float_as_int(q.x) + (__float_as_int(t.x) << 23)),
                       __int_as_float(__float_as_int(q.y) + (__float_as_int(t.y) << 23)));
}
// the largest of three, NaN if one is
__device__ __forceinline__ float max_3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
template <int DT>
__device__ __forceinline__ bool odd_value(uint32_t h) {                        // a 16-bit value that is no number
    constexpr uint32_t E = DT == DT_F16 ? 0x7c00u : 0x7f80u;
    return (h & E) == E;
}

struct Maps {
    CUtensorMap q, k, v;
};

// ---- loader -------------------------------------------------------------------------------------------------------------------
template <int D>
__device__ __forceinline__ void load_role(const AttnArgs& a, const Maps& m, uint8_t* smem, Sync* sy, Walk<kShift> w, int worker, const Shares& shares) {
    using M = Map<D>;
    const int lane = threadIdx.x & 31;
    const int box = min(1 << a.pages.shift, kTileRows), boxes = kTileRows / box, tile_tokens = a.tokens / 2;
    const uint32_t base = smem_u32(smem);
    const uint32_t block_bits = (box == 128 ? 0xffu : (1u << (box >> 4)) - 1u);
    uint32_t c = 0, items = 0;                        // tiles and parts so far
    bool ok = true;
    if (lane == 0) a.joins[worker] = make_int4(0, 0, 0, 0);
    for (;; ++items) {
        Part p;
        p.units = 0;
        if (w.live()) p = part_of(a, w);
        // (every role has done with the item that had the entry before)
        ok = warp_wait(sy, &sy->part_free[items % kParts], ((items / kParts) & 1u) ^ 1u);
        if (!ok) break;
        if (lane < kOddTiles * 4) sy->odd[items % kParts][lane >> 2][lane & 3] = 0;
        __syncwarp();
        if (lane == 0) {
            sy->odd_any[items % kParts] = 0;
            sy->part[items % kParts] = p;
            mbar_arrive(&sy->part_full[items % kParts]);
            if (p.units > 0 && p.whole == 1) {        // (an item that is begun and not finished is the block's last)
                const long long last = shares.begin(worker + 1) - w.until + w.last_unit(a);
                a.joins[worker] = make_int4(shares.worker_of(last) - worker + 1, p.row0, p.tokens * a.group, p.block);
            }
        }
        if (p.units == 0) break;
        const int kv = p.block / a.shared;
        ok = warp_wait(sy, &sy->q_free, (items & 1u) ^ 1u);
        if (!ok) break;
        if (lane == 0) {
            const uint32_t bytes = (uint32_t)(a.group * tile_tokens) * 128u * M::kSubs;
            mbar_arrive_expect_tx(&sy->q_full, bytes * p.tiles);
            for (int t = 0; t < p.tiles; ++t)
                for (int i = 0; i < M::kSubs; ++i)
                    tma_3d(base + M::kQ + t * M::kTile + i * kSubBytes, &m.q, i * 64, p.block * a.group, p.row0 + t * tile_tokens, &sy->q_full);
        }
        auto find = [&](int u) {                      // cache row of this lane's box of key tile u, -1: none
            const int key = p.key0 + (u << kShift) + lane * box;
            int row = -1;
            if (lane < boxes && u < p.units && key <= p.hi && key + box - 1 >= p.lo) {
                row = a.pages.page_row(p.s, key >> a.pages.shift);
                if (row >= 0) row += key & ((1 << a.pages.shift) - 1);
            }
            return row;
        };
        int row = find(0);
        for (int u = 0; u < p.units && ok; ++u, ++c) {
            const int next = find(u + 1);             // (under way while this tile waits for its slot)
            const uint32_t got = __ballot_sync(0xffffffffu, row >= 0);
            const uint32_t bytes = __popc(got) * (uint32_t)box * 128u * M::kSubs;
            if (lane == 0) {
                uint32_t bits = 0;
                for (int b = 0; b < boxes; ++b)
                    if ((got >> b) & 1u) bits |= block_bits << (b * (box >> 4));
                sy->there[c % kSeen] = bits;
            }
#pragma unroll
            for (int kvt = 0; kvt < 2 && ok; ++kvt) {
                const uint32_t n = 2 * c + kvt, slot = n % M::kSlots;
                unsigned long long* const full = kvt ? &sy->v_full[c % kRingBars] : &sy->k_full[c % kRingBars];
                ok = warp_wait(sy, &sy->slot_free[slot], ((n / M::kSlots) & 1u) ^ 1u);
                if (!ok) break;
                if (lane == 0) mbar_arrive_expect_tx(full, bytes);
                __syncwarp();
                if (row >= 0) {
#pragma unroll
                    for (int i = 0; i < M::kSubs; ++i)
                        tma_2d(base + M::kRing + slot * M::kTile + i * kSubBytes + lane * box * 128, kvt ? &m.v : &m.k, kv * D + i * 64, row, full);
                }
                __syncwarp();
            }
            row = next;
        }
        if (!ok) break;
        w.next(a);
    }
    if (!ok) {                                        // copies that are under way land before the block's memory goes
        if (lane == 0) {
            auto landed = [&](unsigned long long* bar, uint32_t parity) {
                const unsigned long long t0 = globaltimer();
                while (!mbar_try_wait(bar, parity) && globaltimer() - t0 < 10000000ull) {}
            };
            if (items > 0) landed(&sy->q_full, (items - 1) & 1u);
            landed(&sy->q_full, items & 1u);
            for (uint32_t n = c > 6 ? c - 6 : 0; n <= c; ++n) {
                landed(&sy->k_full[n % kRingBars], (n / kRingBars) & 1u);
                landed(&sy->v_full[n % kRingBars], (n / kRingBars) & 1u);
            }
        }
        __syncwarp();
    }
}

// ---- products -----------------------------------------------------------------------------------------------------------------
// One warp issues all of a block's products, and what it executes between two of them is time the tensor cores stand still: positions in the rings
// are counted on, not computed, and the two tiles are written out.
__device__ __forceinline__ uint64_t desc_at(uint32_t lo, uint32_t hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
    return d;
}
template <int DT, int D>
struct Products {
    using M = Map<D>;
    static constexpr uint32_t kFmt = DT == DT_F16 ? 0u : 1u;
    // fp32 accumulator, M = 128; S: N = 128, both operands K-major; O: N = D, B MN-major
    static constexpr uint32_t kBasic = (1u << 4) | (kFmt << 7) | (kFmt << 10) | ((128u >> 4) << 24);
    static constexpr uint32_t kIdescS = kBasic | ((128u >> 3) << 17), kIdescO = kBasic | (1u << 16) | (((uint32_t)D >> 3) << 17);
    Sync* sy;
    uint32_t tmem;
    uint32_t lo, hi, vlo;                             // halves of the descriptor of shared memory's first byte, as K-major and as MN-major operand
    bool leader;
    uint32_t kt = 0, vt = 0, kslot = 0, vslot = 1;    // key tiles whose scores (of the first tile), whose P V came last; their slots
    uint32_t sbuf = 0, pbuf = 0;                      // columns of the next scores, of the next P
    uint32_t sdone[2] = {0, 0}, pdone[2] = {0, 0};    // blocks of scores, of P V of each tile
    uint32_t items = 0, outs[2] = {0, 0};

    __device__ __forceinline__ bool key_tile() { return warp_wait(sy, &sy->k_full[kt & (kRingBars - 1)], (kt / kRingBars) & 1u); }
    // S of tile T from the key tile in slot kslot; the last tile of an item moves on to the next key tile
    template <int T, bool LAST>
    __device__ __forceinline__ void scores(bool item_ends) {
        const uint32_t q = lo + ((M::kQ + T * M::kTile) >> 4), k0 = lo + (M::kRing >> 4) + kslot * (M::kTile >> 4);
        if (leader) {
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                const uint32_t off = (k & 3) * 2 + (k >> 2) * (kSubBytes >> 4);
                tc_mma(tmem + sbuf, desc_at(q + off, hi), desc_at(k0 + off, hi), kIdescS, k ? 1u : 0u);
            }
            tc_commit(&sy->s_full[T][sdone[T] & 3u]);
            if (LAST) tc_commit(&sy->slot_free[kslot]);
            if (LAST && item_ends) tc_commit(&sy->q_free);
        }
        __syncwarp();
        ++sdone[T];
        sbuf = sbuf + 128 == M::kScores * 128 ? 0 : sbuf + 128;
        if (LAST) {
            ++kt;
            kslot = kslot + 2 >= M::kSlots ? kslot + 2 - M::kSlots : kslot + 2;
        }
    }
    // O += P V of tile T, the value tile in slot vslot
    template <int T, bool LAST>
    __device__ __forceinline__ bool values(bool first) {
        if (first && !warp_wait(sy, &sy->o_free[T], (outs[T] & 1u) ^ 1u)) return false;       // (the item before has been read)
        if (!warp_wait(sy, &sy->p_full[T][pdone[T] & 3u], (pdone[T] >> 2) & 1u)) return false;
        tc_fence_after();
        const uint32_t v = vlo + (M::kRing >> 4) + vslot * (M::kTile >> 4);
        const uint32_t keep = first ? 0u : 1u;
        if (leader) {
#pragma unroll
            for (int k = 0; k < 8; ++k)                // 16 keys: 8 columns of P, 2048 bytes of V
                mma_ta(tmem + M::kO + D * T, tmem + pbuf + 8 * k, desc_at(v + 128 * k, hi), kIdescO, k ? 1u : keep);
            tc_commit(&sy->pv_done[T][pdone[T] & 3u]);
            if (LAST) tc_commit(&sy->slot_free[vslot]);
        }
        __syncwarp();
        ++pdone[T];
        pbuf = pbuf + 128 == M::kScores * 128 ? 0 : pbuf + 128;
        if (LAST) {
            ++vt;
            vslot = vslot + 2 >= M::kSlots ? vslot + 2 - M::kSlots : vslot + 2;
        }
        return true;
    }
    __device__ __forceinline__ bool value_tile() { return warp_wait(sy, &sy->v_ready[vt & (kRingBars - 1)], (vt / kRingBars) & 1u); }

    // An item of two tiles: the scores of block n + kScores (blocks of both tiles in turns) right behind P V of block n, into the same columns.
    __device__ __forceinline__ bool two(int units) {
        if (!key_tile()) return false;
        tc_fence_after();
        scores<0, false>(false);
        scores<1, true>(units == 1);
        if (M::kScores == 3 && units > 1) {
            if (!key_tile()) return false;
            scores<0, false>(false);
        }
        for (int j = 0; j < units; ++j) {
            if (!value_tile()) return false;
            if (M::kScores == 3) {
                if (!values<0, false>(j == 0)) return false;
                if (j + 1 < units) scores<1, true>(j + 2 == units);
                if (j + 2 < units && !key_tile()) return false;
                if (!values<1, true>(j == 0)) return false;
                if (j + 2 < units) scores<0, false>(false);
            } else {
                if (j + 1 < units && !key_tile()) return false;
                if (!values<0, false>(j == 0)) return false;
                if (j + 1 < units) scores<0, false>(false);
                if (!values<1, true>(j == 0)) return false;
                if (j + 1 < units) scores<1, true>(j + 2 == units);
            }
        }
        return true;
    }
    __device__ __forceinline__ bool one(int units) {
        for (int j = 0; j < M::kScores && j < units; ++j) {
            if (!key_tile()) return false;
            tc_fence_after();
            scores<0, true>(j + 1 == units);
        }
        for (int j = 0; j < units; ++j) {
            const bool more = j + M::kScores < units;
            if (!value_tile() || (more && !key_tile()) || !values<0, true>(j == 0)) return false;
            if (more) scores<0, true>(j + M::kScores + 1 == units);
        }
        return true;
    }
};
template <int DT, int D>
__device__ __forceinline__ void product_role(uint8_t* smem, Sync* sy, uint32_t tmem) {
    const uint64_t d0 = tc_smem_desc(smem_u32(smem));
    Products<DT, D> p;
    p.sy = sy;
    p.tmem = __shfl_sync(0xffffffffu, tmem, 0);       // (the same in all lanes, told so to the compiler: operands in uniform registers)
    p.lo = (uint32_t)d0;
    p.hi = (uint32_t)(d0 >> 32);
    // MN-major: 8-key groups 1024 bytes apart (the descriptor's stride), sub-tiles of 64 columns 16 KB apart (its leading offset)
    p.vlo = D == 64 ? p.lo : p.lo - (1u << 16) + ((uint32_t)(kSubBytes >> 4) << 16);
    p.leader = elect_one();
    Part part;
    for (; next_part(sy, p.items, part); ++p.items) {
        const int units = __shfl_sync(0xffffffffu, part.units, 0), tiles = __shfl_sync(0xffffffffu, part.tiles, 0);
        if (!warp_wait(sy, &sy->q_full, p.items & 1u)) return;
        if (!(tiles == 2 ? p.two(units) : p.one(units))) return;
        ++p.outs[0];
        if (tiles == 2) ++p.outs[1];
        done_part(sy, p.items);
    }
}

// ---- values -------------------------------------------------------------------------------------------------------------------
template <int DT, int D>
__device__ __forceinline__ void value_role(uint8_t* smem, Sync* sy) {
    using M = Map<D>;
    const int lane = threadIdx.x & 31, half = (threadIdx.x >> 5) & 1;
    uint32_t c = 0;
    Part p;
    for (uint32_t items = 0; next_part(sy, items, p); ++items) {
        int lo_all, hi_all, partial = 0;
        seen_by_all(p, 0, p.tokens, lo_all, hi_all);
        const uint32_t mem = items % kParts;
        for (int u = 0; u < p.units; ++u, ++c) {
            const uint32_t slot = (2 * c + 1) % M::kSlots;
            if (!warp_wait(sy, &sy->v_full[c % kRingBars], (c / kRingBars) & 1u)) return;
            const int key0 = p.key0 + (u << kShift);
            const bool some = key0 < lo_all || key0 + 127 > hi_all;          // keys that some token does not see
            const uint32_t there = *(volatile uint32_t*)&sy->there[c % kSeen];
            if (some || there != 0xffu) {
                // a warp has every other four rows: 8 i + 4 half + lane / 8; the other lanes' pieces of 16 bytes
                const int row0 = 4 * half + (lane >> 3);
                const uint32_t tile = smem_u32(smem) + M::kRing + slot * M::kTile + row0 * 128 + (lane & 7) * 16;
                uint32_t none = 0, part = 0;          // bit i: nobody sees the row; some do
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int key = key0 + 8 * i + row0;
                    const bool out = key < p.lo || key > p.hi || !((there >> (i >> 1)) & 1u);
                    none |= (uint32_t)out << i;
                    part |= (uint32_t)(!out && (key < lo_all || key > hi_all)) << i;
                }
                for (uint32_t rows = __reduce_or_sync(0xffffffffu, none); rows; rows &= rows - 1) {
                    const int i = __ffs(rows) - 1;
                    if ((none >> i) & 1u) {
#pragma unroll
                        for (int sub = 0; sub < M::kSubs; ++sub)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + sub * kSubBytes + i * 1024), "r"(0) : "memory");
                    }
                    __syncwarp();
                }
                uint32_t odd = 0;                     // top bit of each 16 bits: an exponent of all ones
                constexpr uint32_t E = DT == DT_F16 ? 0x7c007c00u : 0x7f807f80u, ONE = DT == DT_F16 ? 0x04000400u : 0x00800080u;
                for (uint32_t rows = __reduce_or_sync(0xffffffffu, part); rows; rows &= rows - 1) {
                    const int i = __ffs(rows) - 1;
                    if ((part >> i) & 1u) {
#pragma unroll
                        for (int sub = 0; sub < M::kSubs; ++sub) {
                            uint32_t x[4];
                            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                                         : "r"(tile + sub * kSubBytes + i * 1024) : "memory");
#pragma unroll
                            for (int e = 0; e < 4; ++e) odd |= (x[e] & E) + ONE;
                        }
                    }
                    __syncwarp();
                }
                if (__any_sync(0xffffffffu, odd & 0x80008000u) && partial < kOddTiles) {
                    for (int k = 0; k < 16 * M::kSubs; ++k) {
                        const int i = k & 15;
                        const uint32_t at = tile + (k >> 4) * kSubBytes + i * 1024;
                        if (!((part >> i) & 1u)) continue;
                        uint32_t x[4];
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at) : "memory");
                        bool any = false;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool l = odd_value<DT>(x[e]), h = odd_value<DT>(x[e] >> 16);
                            any |= l || h;
                            x[e] &= (l ? 0u : 0xffffu) | (h ? 0u : 0xffff0000u);
                        }
                        if (any) {
                            const int row = 8 * i + row0;
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
                            atomicOr(&sy->odd[mem][partial][row >> 5], 1u << (row & 31));
                            *(volatile int*)&sy->odd_any[mem] = 1;
                        }
                    }
                }
                partial += some ? 1 : 0;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
            if (lane == 0) mbar_arrive(&sy->v_ready[c % kRingBars]);
        }
        done_part(sy, items);
    }
}

// ---- softmax ------------------------------------------------------------------------------------------------------------------
template <int DT, int D>
__device__ __forceinline__ void softmax_role(const AttnArgs& a, Sync* sy, uint32_t tmem, int worker) {
    using M = Map<D>;
    constexpr float NEG_INF = -__builtin_huge_valf();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = warp >> 2, i = threadIdx.x & 127;     // tile and its row
    const int tile_tokens = a.tokens / 2, my_token = a.token_of(i), my_head = i - my_token * a.group;
    const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16), ocol = tl + M::kO + D * t;
    uint32_t c = 0, seq0 = 0, blocks = 0;
    Part p;
    for (uint32_t items = 0; next_part(sy, items, p); ++items) {
        if (t < p.tiles) {
            const int token = t * tile_tokens + my_token;
            const bool mine = my_token < tile_tokens && token < p.tokens;
            int lo, hi, lo_all, hi_all, lo_any, hi_any, unused;               // keys that this row, every row, some row of the tile sees
            seen_by(p, min(token, p.tokens - 1), lo, hi);
            const int last = min(p.tokens, (t + 1) * tile_tokens);
            seen_by_all(p, t * tile_tokens, last, lo_all, hi_all);
            seen_by(p, t * tile_tokens, lo_any, unused);
            seen_by(p, last - 1, unused, hi_any);
            float m = NEG_INF, l = 0.f;
            bool low = true;                                                   // some row of the warp has no maximum yet
            for (int u = 0; u < p.units; ++u) {
                const uint32_t n = seq0 + (uint32_t)(u * p.tiles + t), buf = n % M::kScores;
                const uint32_t scol = tl + 128 * buf;
                if (!warp_wait(sy, &sy->s_full[t][blocks & 3u], (blocks >> 2) & 1u)) return;
                tc_fence_after();
                const int key0 = p.key0 + (u << kShift);
                const uint32_t there = *(volatile uint32_t*)&sy->there[(c + (uint32_t)u) % kSeen];
                const bool edge = key0 < lo_all || key0 + 127 > hi_all || there != 0xffu;      // keys that some row does not see
                const int from = lo - key0, to = hi - key0;
                float va[32], vb[32];
                // of 32 columns from 32 ch on, the same for all rows: none is seen; every one is
                auto nobody = [&](int ch) { return key0 + ch * 32 > hi_any || key0 + ch * 32 + 31 < lo_any || !((there >> 2 * ch) & 3u); };
                auto hide = [&](int ch, float* v) {                            // those in [from, to], of blocks that are there
                    if (key0 + ch * 32 >= lo_all && key0 + ch * 32 + 31 <= hi_all && ((there >> 2 * ch) & 3u) == 3u) return;
                    const int f = min(max(from - ch * 32, 0), 32), n = min(max(to + 1 - ch * 32, 0), 32);
                    const uint32_t below = n == 32 ? 0xffffffffu : (1u << n) - 1u, front = f == 32 ? 0xffffffffu : (1u << f) - 1u;
                    const uint32_t two = there >> 2 * ch, w = below & ~front & ((two & 1u ? 0xffffu : 0u) | (two & 2u ? 0xffff0000u : 0u));
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[e] = w & (1u << e) ? v[e] : NEG_INF;
                };
                float m4[4] = {NEG_INF, NEG_INF, NEG_INF, NEG_INF};
                if (!edge) {
#pragma unroll 1
                    for (int ch = 0; ch < 4; ch += 2) {
                        tmem_ld32(scol + ch * 32, va);
                        tmem_ld32(scol + ch * 32 + 32, vb);
                        tmem_wait_ld();
                        use32(va);
                        use32(vb);
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            m4[0] = max_3(m4[0], va[e], va[e + 1]); m4[1] = max_3(m4[1], va[e + 2], va[e + 3]);
                            m4[2] = max_3(m4[2], vb[e], vb[e + 1]); m4[3] = max_3(m4[3], vb[e + 2], vb[e + 3]);
                        }
                    }
                } else {
#pragma unroll 1
                    for (int ch = 0; ch < 4; ++ch) {
                        if (nobody(ch)) continue;
                        tmem_ld32(scol + ch * 32, va);
                        tmem_wait_ld();
                        use32(va);
                        hide(ch, va);
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            m4[0] = max_3(m4[0], va[e], va[e + 1]); m4[1] = max_3(m4[1], va[e + 2], va[e + 3]);
                        }
                        __syncwarp();
                    }
                }

                const float mx = max_3(m4[0], m4[1], max_3(m4[2], m4[2], m4[3])) * a.scale2;
                // (a row that sees NaN or an infinite score has no result; said here, since what follows may lose it)
                if (!(mx < -NEG_INF)) l = __int_as_float(0x7fffffff);
                const bool raise = mx > m + kLazy || (m == NEG_INF && mx != NEG_INF);
                if (__any_sync(0xffffffffu, raise)) {
                    const float factor = !raise ? 1.f : m == NEG_INF ? 0.f : ex2(m - mx);
                    if (raise) m = mx;
                    low = __any_sync(0xffffffffu, m == NEG_INF);
                    if (u > 0) {
                        if (!warp_wait(sy, &sy->pv_done[t][(blocks - 1u) & 3u], ((blocks - 1u) >> 2) & 1u)) return;      // O is complete up to here
                        tc_fence_after();
                        l *= factor;
#pragma unroll 1
                        for (int ch = 0; ch < D / 16; ++ch) {
                            float o[16];
                            uint32_t x[16];
                            tc_ld16(ocol + ch * 16, o);
#pragma unroll
                            for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(o[e] * factor);
                            tmem_st16(ocol + ch * 16, x);
                        }
                    }
                }
                const float mm = m == NEG_INF ? 0.f : m;                       // (no key so far: every score is -inf)
                const bool exact = edge || low;                                // (-inf must become 0)
                const float2 scale2 = make_float2(a.scale2, a.scale2), off2 = make_float2(-mm, -mm);
                float2 l4[4] = {};
                // P of 32 columns: of each 16, the pairs of `fma` without the special function units (where every key is seen: a hidden one must be 0)
                auto weigh = [&](int ch, float* v, auto edges) {
                    constexpr bool EDGES = decltype(edges)::value;
                    use32(v);
                    if (EDGES) hide(ch, v);
                    uint32_t x[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const float2 y = fma_2(make_float2(v[e], v[e + 1]), scale2, off2);
                        const float2 q = !EDGES && ((kFmaPairs >> (e >> 1 & 7)) & 1) ? ex2_fma(y) : make_float2(ex2(y.x), ex2(y.y));
                        l4[(e >> 1) & 3] = add_2(l4[(e >> 1) & 3], q);
                        x[e >> 1] = pack16<DT>(q.x, q.y);
                    }
                    tmem_st16(scol + ch * 16, x);
                };
                if (!exact) {
#pragma unroll 1
                    for (int ch = 0; ch < 4; ch += 2) {
                        tmem_ld32(scol + ch * 32, va);
                        tmem_ld32(scol + ch * 32 + 32, vb);                    // (one after the other: 4 x 4096 tokens 389 and 278 us)
                        tmem_wait_ld();
                        use32(vb);
                        weigh(ch, va, Const<false>{});
                        weigh(ch + 1, vb, Const<false>{});
                    }
                } else {
#pragma unroll 1
                    for (int ch = 0; ch < 4; ++ch) {
                        if (nobody(ch)) {
                            uint32_t x[16] = {};
                            tmem_st16(scol + ch * 16, x);
                        } else {
                            tmem_ld32(scol + ch * 32, va);
                            tmem_wait_ld();
                            weigh(ch, va, Const<true>{});
                        }
                        __syncwarp();
                    }
                }
                l += ((l4[0].x + l4[0].y) + (l4[1].x + l4[1].y)) + ((l4[2].x + l4[2].y) + (l4[3].x + l4[3].y));
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sy->p_full[t][blocks & 3u]);                    // S read, P written
                ++blocks;
            }
            // ---- results, or this part's statistics and products
            if (!warp_wait(sy, &sy->pv_done[t][(blocks - 1u) & 3u], ((blocks - 1u) >> 2) & 1u)) return;
            tc_fence_after();
            const bool whole = p.whole == 3;
            const int part_row = token * a.group + my_head;
            const long long slot = (long long)worker * 2 + (p.whole & 1);
            const float inv = l == 0.f ? 0.f : 1.f / l;
            uint16_t* const to = a.out + (long long)(p.row0 + token) * a.ld_out + (p.block * a.group + my_head) * D;
            const bool sectors = ((uintptr_t)a.out & 31) == 0 && a.ld_out % 16 == 0;       // rows of the result start on 32-byte boundaries
            const uint32_t mem = items % kParts;
            const bool odd = *(volatile int*)&sy->odd_any[mem] != 0;
            if (mine && !whole) a.stats[slot * a.part_rows + part_row] = make_float2(l != l ? 0.f : m, l);       // (no result: a maximum that counts)
#pragma unroll 1
            for (int ch = 0; ch < D; ch += 64) {
                float o[64];
                tmem_ld32(ocol + ch, o);
                tmem_ld32(ocol + ch + 32, o + 32);
                tmem_wait_ld();
                use32(o);
                use32(o + 32);
                if (ch == D - 64) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sy->o_free[t]);
                }
                if (odd && mine) {                                             // values that are no numbers, for the tokens that see them
                    int n = 0, alo, ahi;
                    seen_by_all(p, 0, p.tokens, alo, ahi);
                    for (int u = 0; u < p.units; ++u) {
                        const int key0 = p.key0 + (u << kShift);
                        if (!(key0 < alo || key0 + 127 > ahi)) continue;
                        for (int r = 0; r < 128 && n < kOddTiles; ++r) {
                            const int key = key0 + r;
                            const uint32_t bits = *(volatile uint32_t*)&sy->odd[mem][n][r >> 5];
                            if (!((bits >> (r & 31)) & 1u) || key < lo || key > hi) continue;
                            const int first = a.pages.page_row(p.s, key >> a.pages.shift);
                            if (first < 0) continue;
                            const uint16_t* v = a.v + (long long)(first + (key & ((1 << a.pages.shift) - 1))) * a.ld_v + p.block / a.shared * D + ch;
#pragma unroll
                            for (int e = 0; e < 64; ++e) {
                                const uint32_t h = v[e];
                                if (odd_value<DT>(h)) o[e] += unpack16<DT>(h).x;
                            }
                        }
                        ++n;
                    }
                }
                if (mine && whole) {
#pragma unroll
                    for (int k = 0; k < 64; k += 16) {
                        uint32_t x[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = pack16<DT>(o[k + 2 * e] * inv, o[k + 2 * e + 1] * inv);
                        st32B(reinterpret_cast<uint8_t*>(to + ch + k), x, sectors);
                    }
                } else if (mine) {
#pragma unroll
                    for (int k = 0; k < 64; k += 8) {
                        uint32_t x[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = __float_as_uint(o[k + e]);
                        st32B(reinterpret_cast<uint8_t*>(a.part(slot, D, part_row, ch + k)), x, true);
                    }
                }
                __syncwarp();
            }
        }
        seq0 += (uint32_t)(p.units * p.tiles);
        c += (uint32_t)p.units;
        done_part(sy, items);
    }
}

template <int DT, int D>
__global__ void __launch_bounds__(kChunkThreads, 1) attend_chunk(const __grid_constant__ AttnArgs a, const __grid_constant__ Maps m) {
    using M = Map<D>;
    extern __shared__ __align__(1024) uint8_t smem[];
    Sync& sy = *reinterpret_cast<Sync*>(smem + M::kBytes);
    const int warp = threadIdx.x >> 5, worker = blockIdx.x;
    if (threadIdx.x == 0) {
        mbar_init(&sy.q_full, 1);
        mbar_init(&sy.q_free, 1);
        for (int i = 0; i < kRingBars; ++i) {
            mbar_init(&sy.k_full[i], 1);
            mbar_init(&sy.v_full[i], 1);
            mbar_init(&sy.v_ready[i], 2);
        }
        for (int i = 0; i < M::kSlots; ++i) mbar_init(&sy.slot_free[i], 1);
        for (int t = 0; t < 2; ++t) {
            for (int i = 0; i < 4; ++i) {
                mbar_init(&sy.s_full[t][i], 1);
                mbar_init(&sy.p_full[t][i], 4);
                mbar_init(&sy.pv_done[t][i], 1);
            }
            mbar_init(&sy.o_free[t], 4);
        }
        for (int i = 0; i < kParts; ++i) {
            mbar_init(&sy.part_full[i], 1);
            mbar_init(&sy.part_free[i], 8 + 3);       // the warps of the other roles
        }
        sy.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sy.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    wait_for_previous_kernel();
    let_next_kernel_launch();
    Walk<kShift> w;
    // (a key tile for each worker at least: 64 tokens behind 936 14.8 us, 17.0 with shares of an item's beginning more; 4 prompts of 100 12.6 and 12.4)
    const Shares shares = plan<kShift, kChunkThreads>(a, reinterpret_cast<PlanScratch<kChunkThreads>*>(smem), warp == 8 ? worker : 0x7fffffff, kChunkUnit, w);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");              // (copies go where the plan's sums were)
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *(volatile uint32_t*)&sy.tmem;
    if (warp < 8) {
        softmax_role<DT, D>(a, &sy, tmem, worker);
    } else {
        if (warp == 8) load_role<D>(a, m, smem, &sy, w, worker, shares);
        else if (warp == 9) product_role<DT, D>(smem, &sy, tmem);
        else value_role<DT, D>(smem, &sy);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 9) {
        if (*(volatile int*)&sy.abort) __nanosleep(200000);                    // (products that were issued have ended)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess;
        (void)cudaGetLastError();
        return ok ? reinterpret_cast<EncodeTiled>(ptr) : nullptr;
    }();
    return fn;
}
// boxes of 64 columns, 128-byte swizzle, zeros outside
bool encode(CUtensorMap* m, int dtype, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
    const cuuint32_t ones[3] = {1, 1, 1};
    return encode_tiled()(m, dtype == DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, const_cast<void*>(base),
                          dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DT, int D>
cudaError_t launch(const AttnArgs& a, const Maps& m, cudaStream_t stream) {
    constexpr int bytes = Map<D>::kBytes + sizeof(Sync);
    static_assert(bytes <= 232448, "shared memory of a block");
    static SharedMemory allowed;
    const cudaError_t e = allowed.allow((const void*)attend_chunk<DT, D>, bytes);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute pdl;
    pdl.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.workers);
    cfg.blockDim = dim3(kChunkThreads);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = stream;
    cfg.attrs = &pdl;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, attend_chunk<DT, D>, a, m);
}

}  // namespace

cudaError_t launch_chunk(const AttnArgs& a, const mk_paged_cache* c, int heads, cudaStream_t stream) {
    if (!encode_tiled()) return cudaErrorNotSupported;
    Maps m;
    const int D = c->head_dim, box_rows = c->page_size < kTileRows ? c->page_size : kTileRows;
    const cuuint64_t qd[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)a.batch.rows}, qs[2] = {(cuuint64_t)D * 2, (cuuint64_t)a.ld_q * 2};
    const cuuint32_t qb[3] = {64, (cuuint32_t)a.group, (cuuint32_t)(a.tokens / 2)};
    const cuuint64_t cd[2] = {(cuuint64_t)c->kv_heads * D, (cuuint64_t)c->pages * c->page_size}, ks[1] = {(cuuint64_t)a.ld_k * 2}, vs[1] = {(cuuint64_t)a.ld_v * 2};
    const cuuint32_t cb[2] = {64, (cuuint32_t)box_rows};
    const bool empty = c->pages == 0;                  // (then no box is ever asked for)
    if (!encode(&m.q, c->dtype, 3, a.q, qd, qs, qb)) return cudaErrorInvalidValue;
    if (empty) m.k = m.v = m.q;
    else if (!encode(&m.k, c->dtype, 2, a.k, cd, ks, cb) || !encode(&m.v, c->dtype, 2, a.v, cd, vs, cb)) return cudaErrorInvalidValue;
    if (c->dtype == DT_F16) return D == 64 ? launch<DT_F16, 64>(a, m, stream) : launch<DT_F16, 128>(a, m, stream);
    return D == 64 ? launch<DT_BF16, 64>(a, m, stream) : launch<DT_BF16, 128>(a, m, stream);
}

cudaError_t chunk_failures(unsigned* count, cudaStream_t stream) {
    const cudaError_t e = cudaMemcpyFromSymbolAsync(count, g_paged_failed, sizeof(unsigned), 0, cudaMemcpyDeviceToHost, stream);
    return e == cudaSuccess ? cudaStreamSynchronize(stream) : e;
}

}  // namespace mk

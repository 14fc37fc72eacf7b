// How attention over a paged cache is divided among workers, and what its kernels share.
//
// An item is up to `tokens` consecutive new tokens of one sequence and `group` query heads of one kv head: rows token * group + head of one
// operand tile.  (Where more heads share a kv head than the tile has rows, `shared` such blocks of heads read it.)  Its keys are cut into units of
// 2^shift keys.  All units of all items -- in the order sequence, block of heads, tokens -- make one list, which is dealt out evenly by what they
// cost (Cost): each worker has the next N / W of the list's whole cost N, the first N % W one more.  Lengths are known on the device only, so every
// block works out its part itself (about 2 us for up to 128 sequences), and batches of the most unlike lengths load all SMs alike.
// A worker that has an item's units from the first to the last writes results.  Else it leaves the running maximum, the sum and the products of its
// part in the workspace (slot 0: a part that does not begin the item; slot 1: one that begins it); a block joins the parts that its
// own workers have of an item, and a second kernel (paged_attention.cu) those of several blocks, always in the same order.
#pragma once
#include <atomic>

#include "paged.cuh"

namespace mk {

struct AttnArgs {
    Batch batch;
    Pages pages;
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* out;
    long long ld_q, ld_k, ld_v, ld_out;
    int blocks, shared, group, window;                // blocks of `group` heads; blocks that share a kv head
    int group_inverse;                                // 65536 / group + 1: row * group_inverse >> 16 is row / group for rows below 256
    float scale2;                                     // scale * log2(e)
    int tokens;                                       // new tokens of an item
    int align;                                        // an item's first unit begins at a multiple of it, a power of two
    int workers, part_rows;                           // ... and rows of a part in the workspace
    __device__ __forceinline__ int token_of(int row) const { return row * group_inverse >> 16; }
    int4* joins;                                      // of each block: parts of the item that it begins and does not end (0: none), its first
                                                      // row, its rows, its block of heads
    float2* stats;                                    // [block][2][part_rows]: maximum (log2 domain) and sum
    float* parts;                                     // [block][2][head_dim / 8][part_rows][8]: rows side by side, for those who have one each
    __device__ __forceinline__ float* part(long long slot, int head_dim, int row, int col) const {
        return parts + ((slot * (head_dim / 8) + (col >> 3)) * part_rows + row) * 8 + (col & 7);
    }
};

struct Item {
    int lo, hi;                                       // keys some token sees (lo > hi: none)
    int key0, units;                                  // first key of the first unit; units, at least one
};

// (the 64-bit division takes a few hundred cycles, and numbers above 2^32 are rare)
__device__ __forceinline__ long long divide(long long a, long long b) {
    return (unsigned long long)(a | b) >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b);
}
// Shares of the list's cost.
struct Shares {
    long long total, per;
    int workers, longer;                              // `longer` workers have per + 1, the others per
    __device__ __forceinline__ Shares(long long cost, int most, int least) {
        total = cost;
        workers = total ? (int)min((long long)most, max(divide(total, least), 1ll)) : 0;       // (no share below `least`, but of one worker)
        per = workers ? divide(total, workers) : 0;
        longer = (int)(total - per * workers);
    }
    __device__ __forceinline__ long long begin(int w) const { return w * per + min(w, longer); }
    __device__ __forceinline__ int worker_of(long long at) const {
        const long long border = (per + 1) * longer;
        return (int)(at < border ? divide(at, per + 1) : longer + divide(at - border, per));
    }
};

// Costs of the chunk kernel: an item's beginning and end, a key tile with both query tiles, with one.  (Key tiles alone, all alike: 4 x 4096 tokens 433
// instead of 413 us for 64-wide heads, 311 instead of 283 for 128-wide, 24 sequences of up to 700 tokens with a window 125 instead of 115.)
constexpr int kChunkBegin = 4, kChunkUnit = 3, kChunkHalf = 2;

// What an item costs: its beginning and end, and each of its units.  A place in the list of costs is the first unit whose end lies behind it.
struct Cost {
    int begin, unit;
    __device__ __forceinline__ long long of(int units) const { return begin + (long long)units * unit; }
    __device__ __forceinline__ int unit_at(long long at, int units) const {            // at: from the item's beginning on
        if (unit == 1) return (int)min(max(at - begin, 0ll), (long long)units);
        return (int)min(max(divide(max(at - begin, 0ll) + unit - 1, unit), 0ll), (long long)units);
    }
};

template <int SHIFT>
__device__ __forceinline__ Item item_at(const AttnArgs& a, long long p0, int tokens) {
    const long long cap = a.pages.capacity();
    Item it;
    it.hi = (int)min(max(p0 + tokens - 1, -1ll), cap - 1);
    it.lo = a.window > 0 ? (int)min(max(p0 + 1 - a.window, 0ll), cap) : 0;
    it.key0 = it.hi < it.lo ? 0 : it.lo & -a.align;
    it.units = it.hi < it.lo ? 1 : ((it.hi - it.key0) >> SHIFT) + 1;
    return it;
}

template <int SHIFT>
__device__ __forceinline__ Cost cost_of(const AttnArgs& a, int tokens) {
    if (SHIFT < 7) return Cost{0, 1};                 // (few rows: a unit is a unit)
    return Cost{kChunkBegin, tokens > a.tokens / 2 ? kChunkUnit : kChunkHalf};
}
template <int SHIFT>
__device__ __forceinline__ long long item_cost(const AttnArgs& a, long long p0, int tokens) {
    return cost_of<SHIFT>(a, tokens).of(item_at<SHIFT>(a, p0, tokens).units);
}
// cost of one block of heads of sequence s, its items first, first + step, ...
template <int SHIFT>
__device__ __forceinline__ long long sequence_cost(const AttnArgs& a, int s, int first = 0, int step = 1) {
    const int r0 = a.batch.first(s), n = a.batch.count(s, r0);
    if (n == 0) return 0;
    const long long p = a.batch.position(s);
    long long sum = 0;
    for (long long t = (long long)first * a.tokens; t < n; t += (long long)step * a.tokens)
        sum += item_cost<SHIFT>(a, p + t, (int)min((long long)a.tokens, n - t));
    return sum;
}

// A worker's way through the list, from item to item.
template <int SHIFT>
struct Walk {
    int s, kv, t;                                     // sequence, block of heads, first token of the item in the sequence
    int r0, n;                                        // rows of the sequence
    long long p;                                      // its position
    int unit, stop;                                   // the worker's units of the item
    long long until;                                  // where the worker's share ends, from the item's beginning on
    Item item;

    __device__ __forceinline__ bool live() const { return unit < stop; }
    __device__ __forceinline__ int item_tokens(const AttnArgs& a) const { return min(a.tokens, n - t); }
    __device__ __forceinline__ Cost cost(const AttnArgs& a) const { return cost_of<SHIFT>(a, item_tokens(a)); }
    // the share goes on behind this item
    __device__ __forceinline__ bool goes_on(const AttnArgs& a) const { return until > cost(a).of(item.units); }
    // place of the item's last unit, from its beginning on: whose share begins at or in front of it has that unit, or one in front
    __device__ __forceinline__ long long last_unit(const AttnArgs& a) const { return cost(a).of(item.units - 1); }
    __device__ __forceinline__ void sequence(const AttnArgs& a, int seq) {
        s = seq;
        r0 = a.batch.first(s);
        n = a.batch.count(s, r0);
        p = a.batch.position(s);
    }
    __device__ __forceinline__ void enter(const AttnArgs& a, long long at) {
        item = item_at<SHIFT>(a, p + t, item_tokens(a));
        const Cost c = cost(a);
        unit = at > 0 ? c.unit_at(at, item.units) : 0;
        stop = until >= c.of(item.units) ? item.units : c.unit_at(until, item.units);
    }
    // to place `at` of the sequence's list (a block of heads costs `per`), with a share of `length`.  All lanes of a warp;
    // where items are many each lane looks at one (one after the other, here and for the sums: 4 x 4096 tokens 397 us instead of 390)
    __device__ __forceinline__ void start(const AttnArgs& a, int seq, long long at, long long per, long long length) {
        sequence(a, seq);
        kv = (int)divide(at, per);
        at -= kv * per;
        const int lane = threadIdx.x & 31;
        t = 0;
        if (n < 8 * a.tokens) {                       // (few items: one after the other)
            for (;; t += a.tokens) {
                const long long c = item_cost<SHIFT>(a, p + t, item_tokens(a));
                if (at < c || t + a.tokens >= n) break;
                at -= c;
            }
        } else {
            long long base = 0;                       // first token of lane 0's item
            for (;;) {
                const long long mine = base + (long long)lane * a.tokens;
                long long run = mine < n ? item_cost<SHIFT>(a, p + mine, (int)min((long long)a.tokens, n - mine)) : 0;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const long long up = __shfl_up_sync(0xffffffffu, run, d);
                    if (lane >= d) run += up;
                }
                int in = __popc(__ballot_sync(0xffffffffu, run <= at));                    // items in front of it
                if (in == 32 && base + 32ll * a.tokens < n) {
                    base += 32ll * a.tokens;
                    at -= __shfl_sync(0xffffffffu, run, 31);
                    continue;
                }
                in = min(in, (int)(n - 1 - base) / a.tokens);
                const long long front = __shfl_sync(0xffffffffu, run, max(in - 1, 0));
                if (in > 0) at -= front;
                base += (long long)in * a.tokens;
                break;
            }
            t = (int)base;
        }
        until = at + length;
        enter(a, at);
        if (unit == item.units) next(a);              // (the share begins behind the item's last unit)
    }
    // to the next item
    __device__ __forceinline__ void next(const AttnArgs& a) {
        until -= cost(a).of(item.units);
        unit = stop = 0;
        if (until <= 0) return;
        t += a.tokens;
        if (t >= n) {
            t = 0;
            if (++kv == a.blocks) {
                kv = 0;
                do sequence(a, s + 1);
                while (n == 0 && s + 1 < a.batch.seqs);
            }
        }
        enter(a, 0);
    }
};

template <int THREADS>
struct PlanScratch {
    long long sums[THREADS / 32];
    long long ends[THREADS];                          // inclusive sums of a round's sequences
};

// Every thread of the block calls it with its warp's worker.  Returns how the list is dealt out, at least `least` to a worker (no less than a
// unit, so that a share inside an item has one); `walk` is at the worker's first unit, if it has any.
template <int SHIFT, int THREADS>
__device__ __forceinline__ Shares plan(const AttnArgs& a, PlanScratch<THREADS>* sc, int worker, int least, Walk<SHIFT>& walk) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    if (a.batch.seqs <= 128) {                        // a few sequences a lane: every warp by itself, in 32 bits
        const int each = (a.batch.seqs + 31) / 32;
        int cost[4], run = 0;
        bool big = false;
        long long only = 0;                           // where each lane has a sequence at most and items are many: lanes share one
        const bool share = SHIFT >= 7 && a.batch.seqs <= 16 && a.batch.rows / 8 >= a.batch.seqs * a.tokens;
        if (share) {
            const int log = a.batch.seqs > 1 ? __clz(a.batch.seqs - 1) - 27 : 5;       // 2^log lanes of a sequence
            const int s = lane >> log;
            only = s < a.batch.seqs ? sequence_cost<SHIFT>(a, s, lane & ((1 << log) - 1), 1 << log) : 0;
            for (int d = 1; d < 1 << log; d <<= 1) only += __shfl_xor_sync(0xffffffffu, only, d);
            only = __shfl_sync(0xffffffffu, only, (lane << log) & 31);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int s = lane * each + k;
            const long long c = k < each && s < a.batch.seqs ? (share ? only : sequence_cost<SHIFT>(a, s)) : 0;
            big |= c > (1 << 23) / a.blocks;          // (128 of them stay below 2^30)
            cost[k] = (int)c * a.blocks;
            run += cost[k];
        }
        if (!__any_sync(0xffffffffu, big)) {
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, run, d);
                if (lane >= d) run += up;
            }
            const Shares shares(__shfl_sync(0xffffffffu, run, 31), a.workers, least);
            walk.unit = walk.stop = 0;
            if (worker < shares.workers) {
                const int begin = (int)shares.begin(worker);
                const int in = __popc(__ballot_sync(0xffffffffu, run <= begin));       // the lane that has it
                int at = begin - (in > 0 ? __shfl_sync(0xffffffffu, run, in - 1) : 0), k = 0, c = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int u = __shfl_sync(0xffffffffu, cost[i], in);
                    if (k == i) {
                        c = u;
                        if (at >= u) { at -= u; ++k; }
                    }
                }
                walk.start(a, in * each + k, at, c / a.blocks, shares.begin(worker + 1) - begin);
            }
            return shares;
        }
    }
    const int rounds = (a.batch.seqs + THREADS - 1) / THREADS;
    long long mine = 0, sum = 0;
    for (int r = 0; r < rounds; ++r) {
        const int s = r * THREADS + t;
        mine = s < a.batch.seqs ? sequence_cost<SHIFT>(a, s) * a.blocks : 0;
        sum += mine;
    }
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) sc->sums[warp] = sum;
    __syncthreads();
    long long total = 0;
    for (int w = 0; w < THREADS / 32; ++w) total += sc->sums[w];
    const Shares shares(total, a.workers, least);
    const bool mine_too = worker < shares.workers;
    const long long begin = mine_too ? shares.begin(worker) : total;
    walk.unit = walk.stop = 0;
    long long base = 0;
    for (int r = 0; r < rounds; ++r) {
        if (rounds > 1) {
            const int s = r * THREADS + t;
            mine = s < a.batch.seqs ? sequence_cost<SHIFT>(a, s) * a.blocks : 0;
        }
        long long run = mine;
        for (int d = 1; d < 32; d <<= 1) {
            const long long up = __shfl_up_sync(0xffffffffu, run, d);
            if (lane >= d) run += up;
        }
        __syncthreads();                              // (the previous round's sums have been read)
        if (lane == 31) sc->sums[warp] = run;
        __syncthreads();
        long long before = base, all = 0;
        for (int w = 0; w < THREADS / 32; ++w) {
            if (w < warp) before += sc->sums[w];
            all += sc->sums[w];
        }
        sc->ends[t] = before + run;
        __syncthreads();
        if (mine_too && begin >= base && begin < base + all) {
            int at = 0;                               // sequences of the round that end at or in front of `begin`
            for (int i = lane; i < THREADS; i += 32) at += sc->ends[i] <= begin;
            for (int d = 16; d; d >>= 1) at += __shfl_xor_sync(0xffffffffu, at, d);
            const long long first = at > 0 ? sc->ends[at - 1] : base;
            walk.start(a, r * THREADS + at, begin - first, divide(sc->ends[at] - first, a.blocks), shares.begin(worker + 1) - begin);
        }
        base += all;
    }
    return shares;
}

// Joins `count` parts of rows [row_begin, row_end) of an item, ROWS of them: part i has slot(i).  With M the largest of their maxima m_i
//   l = sum_i 2^(m_i - M) l_i,   o = sum_i 2^(m_i - M) o_i,   always in the same order.
// A thread has eight columns of a row; where that leaves threads over they share a row's parts and add through shared memory.  What a thread waits for
// is memory, so it asks for kAtOnce parts together: two, as most items have; four take half as many threads again in registers (4 x 4096 tokens 402 us
// instead of 399, a prompt of 2000 50 instead of 46), one after the other one sequence of 16384 keys 17 instead of 16.  All threads of the block call it.  write(row, column, l, o) takes eight columns.
template <int D, int ROWS, int THREADS>
struct Join {
    static constexpr int kTasks = ROWS * (D / 8), kSplits = THREADS / kTasks, kAtOnce = 2;
    static_assert(kSplits * kTasks == THREADS, "threads of a join");
    float o[kSplits > 1 ? 8 : 1][kSplits > 1 ? THREADS : 1];
    float m[kSplits > 1 ? THREADS : 1], l[kSplits > 1 ? THREADS : 1];

    static __device__ __forceinline__ float factor(float m, float to) { return m == to ? 1.f : ex2(m - to); }      // (-inf: 0, unless both are)

    template <class Slot, class Write>
    __device__ __forceinline__ void run(const AttnArgs& a, int count, int row_begin, int row_end, Slot slot, Write write) {
        constexpr float NEG_INF = -__builtin_huge_valf();
        const int t = threadIdx.x, split = t / kTasks, row = row_begin + t % ROWS, col = t % kTasks / ROWS * 8;
        const bool mine = row < row_end;
        float mx = NEG_INF, sum = 0.f, x[8] = {};
        for (int i = split; mine && i < count; i += kSplits * kAtOnce) {
            float2 st[kAtOnce];
            float4 v[kAtOnce][2];
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                st[k] = make_float2(NEG_INF, 0.f);
                v[k][0] = v[k][1] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i + k * kSplits < count) {
                    const long long at = slot(i + k * kSplits);
                    const float4* const src = reinterpret_cast<const float4*>(a.part(at, D, row, col));
                    st[k] = __ldcg(&a.stats[at * a.part_rows + row]);
                    v[k][0] = __ldcg(src);
                    v[k][1] = __ldcg(src + 1);
                }
            }
            float to = mx;
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) to = fmaxf(to, st[k].x);
            if (to == NEG_INF) continue;              // (none of them saw a key)
            const float f = factor(mx, to);
            sum *= f;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= f;
            mx = to;
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                if (st[k].x == NEG_INF) continue;     // (nothing to add)
                const float g = factor(st[k].x, to);
                sum += g * st[k].y;
                x[0] += g * v[k][0].x; x[1] += g * v[k][0].y; x[2] += g * v[k][0].z; x[3] += g * v[k][0].w;
                x[4] += g * v[k][1].x; x[5] += g * v[k][1].y; x[6] += g * v[k][1].z; x[7] += g * v[k][1].w;
            }
        }
        if (kSplits > 1) {
            m[t] = mx;
            l[t] = sum;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e][t] = x[e];
            __syncthreads();
            if (split > 0 || !mine) return;
            float to = mx;
            for (int k = 1; k < kSplits; ++k) to = fmaxf(to, m[t + k * kTasks]);
            if (to != NEG_INF) {
                const float f = factor(mx, to);
                sum *= f;
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] *= f;
                for (int k = 1; k < kSplits; ++k) {
                    const int at = t + k * kTasks;
                    if (m[at] == NEG_INF) continue;
                    const float g = factor(m[at], to);
                    sum += g * l[at];
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] += g * o[e][at];
                }
            }
        }
        if (mine) write(row, col, sum, make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]));
    }
};

// eight columns of an item's row (of `a.group` heads a token) of the result
template <int DT, int D>
__device__ __forceinline__ void write_result(const AttnArgs& a, int row0, int block, int row, int col, float l, const float4& x, const float4& y) {
    const float inv = l == 0.f ? 0.f : 1.f / l;       // (no key: zeros)
    const int tok = a.token_of(row);
    uint16_t* to = a.out + (long long)(row0 + tok) * a.ld_out + (block * a.group + row - tok * a.group) * D + col;
    *reinterpret_cast<uint4*>(to) = make_uint4(pack16<DT>(x.x * inv, x.y * inv), pack16<DT>(x.z * inv, x.w * inv),
                                               pack16<DT>(y.x * inv, y.y * inv), pack16<DT>(y.z * inv, y.w * inv));
}

// items of few rows (paged_attention_few.cu): rows of an item, workers of a block
constexpr int kFewRows = 16;
constexpr int kFewWarps = 8;
cudaError_t launch_few(const AttnArgs& a, float* own /* [worker][kFewRows][head_dim] */, int head_dim, int dtype, int blocks, cudaStream_t stream);

// items of up to 256 rows, a positive scale (paged_attention_chunk.cu): two tiles of 128 rows, a worker per block
constexpr int kChunkTile = 128;
cudaError_t launch_chunk(const AttnArgs& a, const mk_paged_cache* cache, int heads, cudaStream_t stream);
cudaError_t chunk_failures(unsigned* count, cudaStream_t stream);

// A kernel's shared memory beyond 48 KB, asked for once per device.
struct SharedMemory {
    std::atomic<unsigned long long> devices{0};
    cudaError_t allow(const void* kernel, int bytes) {
        int device = 0;
        cudaError_t e = cudaGetDevice(&device);
        const unsigned long long bit = 1ull << (device & 63);
        if (e != cudaSuccess || (device < 64 && (devices.load(std::memory_order_relaxed) & bit))) return e;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess && device < 64) devices.fetch_or(bit, std::memory_order_relaxed);
        return e;
    }
};

__device__ __forceinline__ void let_next_kernel_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace mk

// Attention over a paged cache for items of at most 16 rows (new tokens x heads of a group): single tokens, a few speculative ones.
//
// Bound by memory: K and V are read once (heads of a group and tokens of a sequence share them), 2 * 2 * head_dim bytes a key, for 4 * 16 * head_dim
// products, far below what warp-level matrix instructions give.  Measured: 64 sequences of 1 to 4096 keys, bf16, 4 kv heads of 128: 57 us, 77 % of the
// measured copy rate; short of that by what comes before and after the keys, 8 to 10 us (launches, the plan, the first look-ups, the joins):
// one sequence of 1024 keys 9.1 us, of 16384 15.7.  So every warp is a worker of its own (paged_attention.cuh): it
// copies units of 8 KB (16 keys of head_dim 128, 32 of 64) into its own ring of three with 16-byte asynchronous copies, which follow the
// page table row by row and write zeros for keys that are not there, and meets no other warp.  16 rows x unit:
//   S = Q K^T   mma m16n8k16, K rows through ldmatrix (16-byte pieces swizzled by row: no bank conflicts), fp32
//   P = 2^(S scale log2(e) - m), rounded to the operand type, in registers the A operand of
//   O += P V    V through transposing ldmatrix
// P is rounded to the second product's operand type; sums of weights are of the unrounded ones, everything else is fp32.  Items of at most 8 rows: the
// operand's other 8 rows take what the rounding left over, so that 16 bits more of P count, at no cost (64 ragged sequences 56.7 us with and without,
// one of 1024 keys 9.1); nothing else is done for them (8 kv heads of 64: 63.5 us instead of 65.3).  Items of 16 rows would need products of their own for it.
// The maximum is only raised when it grows by more than 2^8, so that O is seldom scaled.
#include "mma.cuh"
#include "paged_attention.cuh"

namespace mk {
namespace {

constexpr int kStagesFew = 3;
constexpr int kUnitBytes = 8192;                      // K and V of a unit
constexpr float kRaise = 8.0f;
// Units that a worker has at least, where there are few: one sequence of 1024 keys 9.4 us with one, 11.4 with two, 13.6 with four.
constexpr int kLeastUnits = 1;

struct Piece {                                        // a part that a warp has of an item (rows 0: none)
    int rows, row0, block;
    int last;                                         // of one that begins the item and does not end it: the worker that does
    bool ends;                                        // it ends the item
    bool far;                                         // its products are in the workspace, not in the warp's ring
};

template <int D> constexpr int unit_shift = D == 128 ? 4 : 5;

__device__ __forceinline__ void copy16_or_zero(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

template <int DT>
__device__ __forceinline__ void mma16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if (DT == DT_F16) mma_f16(c, a, b0, b1);
    else mma_bf16(c, a, b0, b1);
}
// infinity or NaN in one of two 16-bit values
template <int DT>
__device__ __forceinline__ bool not_finite(uint32_t w) {
    constexpr uint32_t E = DT == DT_F16 ? 0x7c00u : 0x7f80u;
    return (w & E) == E || ((w >> 16) & E) == E;
}

// HALVES: 1 for items of at most 8 rows (the matrix instruction's other 8 are zeros in Q and what P lost to rounding in the second product), else 2
template <int DT, int D, int HALVES>
__global__ void __launch_bounds__(kFewWarps * 32, 1) attend_few(const __grid_constant__ AttnArgs a, float* own) {
    constexpr int SHIFT = unit_shift<D>, U = 1 << SHIFT, NT = U / 8, KS = U / 16, DK = D / 16, DN = D / 8;
    constexpr int CH = D / 8, ROWS_PER_COPY = 32 / CH;          // 16-byte pieces of a row; rows that 32 lanes copy
    constexpr float NEG_INF = -__builtin_huge_valf();
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ PlanScratch<kFewWarps * 32> scratch;
    wait_for_previous_kernel();
    let_next_kernel_launch();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, worker = blockIdx.x * kFewWarps + warp;
    Walk<SHIFT> w;
    const Shares shares = plan<SHIFT, kFewWarps * 32>(a, &scratch, worker, kLeastUnits, w);
    if (threadIdx.x == 0) a.joins[blockIdx.x] = make_int4(0, 0, 0, 0);
    __shared__ Piece pieces[kFewWarps][2];
    __shared__ float2 stats[kFewWarps][2][kFewRows];
    if (lane < 2) pieces[warp][lane].rows = 0;
    float* const near = reinterpret_cast<float*>(smem + warp * (kStagesFew * kUnitBytes));
    __syncwarp();
    const uint32_t ring = smem_u32(smem) + warp * (kStagesFew * kUnitBytes);
    const int quad = lane >> 2, pair = (lane & 3) * 2;           // this thread's rows quad, quad + 8; columns pair, pair + 1 of each 8

    while (w.live()) {
        const int tokens = w.item_tokens(a), rows = tokens * a.group, u0 = w.unit;
        const int count = w.stop - u0, base_row = w.r0 + w.t, kv = w.kv, s = w.s;
        const Item it = w.item;
        const long long p0 = w.p + w.t;
        const int first_key = it.key0 + (u0 << SHIFT);
        // keys that this thread's rows see
        int lo_r[HALVES], hi_r[HALVES];
#pragma unroll
        for (int i = 0; i < HALVES; ++i) {
            const long long p = p0 + a.token_of(quad + 8 * i);
            hi_r[i] = (int)min(max(p, -1ll), (long long)it.hi);
            lo_r[i] = a.window > 0 ? (int)min(max(p + 1 - a.window, 0ll), 0x7fffffffll) : 0;
        }
        const int hi_all = (int)min(max(p0, -1ll), (long long)it.hi);                              // keys that every row sees
        const int lo_all = a.window > 0 ? (int)min(max(p0 + tokens - a.window, 0ll), 0x7fffffffll) : 0;

        // ---- the page table, 32 blocks of 16 keys at a time, a block per lane
        int block0 = first_key >> 4, held = -1;
        auto hold = [&](int at) {
            block0 = at;
            const int key = (at + lane) << 4;
            held = -1;
            if ((at + lane) >= 0 && key <= it.hi) {
                const int f = a.pages.page_row(s, key >> a.pages.shift);
                if (f >= 0) held = f + (key & ((1 << a.pages.shift) - 1));
            }
        };
        hold(block0);
        // ---- Q fragments
        uint32_t q[DK][4];
        long long row_at[HALVES];                                // this thread's rows of the packed batch, -1: none
#pragma unroll
        for (int k = 0; k < DK; ++k) q[k][1] = q[k][3] = 0u;
#pragma unroll
        for (int i = 0; i < HALVES; ++i) {
            const int row = quad + 8 * i, tok = a.token_of(row);
            row_at[i] = row < rows ? (long long)(base_row + tok) : -1;
            const uint16_t* src = a.q + row_at[i] * a.ld_q + (kv * a.group + row - tok * a.group) * D + pair;
#pragma unroll
            for (int k = 0; k < DK; ++k) {
                q[k][i] = row < rows ? __ldg(reinterpret_cast<const uint32_t*>(src + k * 16)) : 0u;
                q[k][i + 2] = row < rows ? __ldg(reinterpret_cast<const uint32_t*>(src + k * 16 + 8)) : 0u;
            }
        }
        uint32_t absent = 0;                                     // two bits of unit u from bit 2 (u % 16): blocks that are not there
        const uint16_t* kp = a.k + kv / a.shared * D + (lane % CH) * 8;
        const uint16_t* vp = a.v + kv / a.shared * D + (lane % CH) * 8;
        auto request = [&](int u) {                              // unit u of this part
            if (u < count) {
                const int key0 = first_key + (u << SHIFT);
                if ((key0 >> 4) + U / 16 > block0 + 32) hold(key0 >> 4);
                const uint32_t stage = ring + (u % kStagesFew) * kUnitBytes;
                uint32_t gone = 0;
#pragma unroll
                for (int b = 0; b < U / 16; ++b) {
                    const int f = __shfl_sync(0xffffffffu, held, (key0 >> 4) + b - block0);
                    gone |= (f < 0 ? 1u : 0u) << b;
#pragma unroll
                    for (int i = 0; i < 16 / ROWS_PER_COPY; ++i) {
                        const int row = i * ROWS_PER_COPY + lane / CH, key = key0 + b * 16 + row;
                        const bool there = f >= 0 && key >= it.lo && key <= it.hi;
                        const long long at = there ? f + row : 0;
                        const uint32_t to = stage + (b * 16 + row) * (D * 2) + (((lane % CH) ^ (row & 7)) << 4);
                        copy16_or_zero(to, kp + at * a.ld_k, there);
                        copy16_or_zero(to + kUnitBytes / 2, vp + at * a.ld_v, there);
                    }
                }
                absent = (absent & ~(3u << 2 * (u & 15))) | gone << 2 * (u & 15);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };

        float o[DN][4];
#pragma unroll
        for (int i = 0; i < DN; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
        float m[HALVES], l[HALVES];
#pragma unroll
        for (int i = 0; i < HALVES; ++i) { m[i] = NEG_INF; l[i] = 0.f; }
        for (int u = 0; u < kStagesFew - 1; ++u) request(u);
        for (int u = 0; u < count; ++u) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kStagesFew - 2) : "memory");
            __syncwarp();                                        // ... of every lane; and all have read the stage that is requested next
            request(u + kStagesFew - 1);
            const uint32_t ks = ring + (u % kStagesFew) * kUnitBytes, vs = ks + kUnitBytes / 2;
            const int key0 = first_key + (u << SHIFT);
            float sc[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
                const int row = n * 8 + (lane & 7);
#pragma unroll
                for (int k = 0; k < DK; k += 2) {
                    uint32_t b[4];
                    ldmatrix_x4(ks + row * (D * 2) + (((k * 2 + (lane >> 3)) ^ (row & 7)) << 4), b[0], b[1], b[2], b[3]);
                    mma16<DT>(sc[n], q[k], b[0], b[1]);
                    mma16<DT>(sc[n], q[k + 1], b[2], b[3]);
                }
            }
            const bool partial = key0 < lo_all || key0 + U - 1 > hi_all;      // keys that some row does not see
            const uint32_t gone = (absent >> 2 * (u & 15)) & 3u;
            float mx[HALVES];
#pragma unroll
            for (int i = 0; i < HALVES; ++i) mx[i] = NEG_INF;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int e = 0; e < 2 * HALVES; ++e) sc[n][e] *= a.scale2;
                if (partial || gone) {
                    const bool here = !((gone >> (n / 2)) & 1u);
                    const int key = key0 + n * 8 + pair;
#pragma unroll
                    for (int e = 0; e < 2 * HALVES; ++e) {
                        const int j = key + (e & 1);
                        if (!here || j < lo_r[e >> 1] || j > hi_r[e >> 1]) sc[n][e] = NEG_INF;
                    }
                }
#pragma unroll
                for (int i = 0; i < HALVES; ++i) mx[i] = fmaxf(mx[i], fmaxf(sc[n][2 * i], sc[n][2 * i + 1]));
            }
            bool raise = false;
#pragma unroll
            for (int i = 0; i < HALVES; ++i) {
                mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
                mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
                raise |= mx[i] > m[i] + kRaise || (m[i] == NEG_INF && mx[i] > NEG_INF);
            }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int i = 0; i < HALVES; ++i) {
                    const float to = fmaxf(m[i], mx[i]), f = m[i] == NEG_INF ? 0.f : ex2(m[i] - to);
                    m[i] = to;
                    l[i] *= f;
#pragma unroll
                    for (int n = 0; n < DN; ++n) {
                        o[n][2 * i] *= f;
                        o[n][2 * i + 1] *= f;
                        if (HALVES == 1) {
                            o[n][2] *= f;
                            o[n][3] *= f;
                        }
                    }
                }
            }
            uint32_t p[KS][4] = {};
#pragma unroll
            for (int i = 0; i < HALVES; ++i) {
                const float off = m[i] == NEG_INF ? 0.f : m[i];   // (no key so far: every score is -inf)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float a0 = ex2(sc[n][2 * i] - off), a1 = ex2(sc[n][2 * i + 1] - off);
                    l[i] += a0 + a1;
                    const uint32_t high = pack16<DT>(a0, a1);
                    p[n >> 1][(n & 1) * 2 + i] = high;
                    if (HALVES == 1) {
                        const float2 h = unpack16<DT>(high);
                        p[n >> 1][(n & 1) * 2 + 1] = pack16<DT>(a0 - h.x, a1 - h.y);
                    }
                }
            }
            // a value that is no number must not reach the tokens that do not see its key through 0 * it
            bool odd = false;
            if (partial && tokens > 1) {
                for (int i = lane; i < U * CH; i += 32) {
                    uint32_t x[4];
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(vs + i * 16) : "memory");
                    odd |= not_finite<DT>(x[0]) || not_finite<DT>(x[1]) || not_finite<DT>(x[2]) || not_finite<DT>(x[3]);
                }
                odd = __any_sync(0xffffffffu, odd);
            }
#pragma unroll
            for (int k = 0; k < KS; ++k) {
#pragma unroll
                for (int n = 0; n < DN; n += 2) {
                    const int row = k * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
                    uint32_t b[4];
                    ldmatrix_x4_trans(vs + row * (D * 2) + (((n + (lane >> 4)) ^ (row & 7)) << 4), b[0], b[1], b[2], b[3]);
                    if (!odd) {
                        mma16<DT>(o[n], p[k], b[0], b[1]);
                        mma16<DT>(o[n + 1], p[k], b[2], b[3]);
                        continue;
                    }
                    for (int t = 0; t < tokens; ++t) {           // token by token, its rows and the values it sees
                        const long long at = p0 + t;
                        const int hi = (int)min(max(at, -1ll), (long long)it.hi);
                        const int lo = a.window > 0 ? (int)min(max(at + 1 - a.window, 0ll), 0x7fffffffll) : 0;
                        const bool r0 = a.token_of(quad) == t, r1 = HALVES == 2 ? a.token_of(quad + 8) == t : r0;
                        uint32_t bt[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int key = key0 + k * 16 + (e & 1) * 8 + pair;
                            bt[e] = b[e] & ((key >= lo && key <= hi ? 0xffffu : 0u) | (key + 1 >= lo && key + 1 <= hi ? 0xffff0000u : 0u));
                        }
                        float c[2][4] = {};
                        mma16<DT>(c[0], p[k], bt[0], bt[1]);
                        mma16<DT>(c[1], p[k], bt[2], bt[3]);
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (e & 2 ? r1 : r0) o[n + (e >> 2)][e & 3] += c[e >> 2][e & 3];
                    }
                }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();                                            // the ring is free for the next part
#pragma unroll
        for (int i = 0; i < HALVES; ++i) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        }
        if (HALVES == 1) {                                       // (where a value is infinite the low half's sum may be of the other sign: left out)
#pragma unroll
            for (int n = 0; n < DN; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (fabsf(o[n][e]) < -NEG_INF) o[n][e] += o[n][e + 2];
        }
        // ---- results, or this part's statistics and products
        const bool whole = u0 == 0 && count == it.units;
        // (the worker's last part has the ring to itself; one in front of others, of which there is one at most, goes to the workspace)
        const bool far = w.goes_on(a);
        if (!whole && lane == 0) {
            // (an item that is begun and not finished is the worker's last)
            const bool ends = u0 + count == it.units;
            const int last = ends || u0 > 0 ? 0 : shares.worker_of(shares.begin(worker + 1) - w.until + w.last_unit(a));
            pieces[warp][u0 == 0 ? 1 : 0] = Piece{rows, base_row, kv, last, ends, far};
        }
#pragma unroll
        for (int i = 0; i < HALVES; ++i) {
            const int row = quad + 8 * i;
            if (row >= rows) continue;
            if (whole) {
                const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
                uint16_t* to = a.out + row_at[i] * a.ld_out + (kv * a.group + row - a.token_of(row) * a.group) * D + pair;
#pragma unroll
                for (int n = 0; n < DN; ++n) *reinterpret_cast<uint32_t*>(to + n * 8) = pack16<DT>(o[n][2 * i] * inv, o[n][2 * i + 1] * inv);
            } else {
                // (no result: a maximum that counts)
                if ((lane & 3) == 0) stats[warp][u0 == 0 ? 1 : 0][row] = make_float2(l[i] != l[i] ? 0.f : m[i], l[i]);
                float* const to = (far ? own + (long long)worker * kFewRows * D : near) + row * D + pair;
#pragma unroll
                for (int n = 0; n < DN; ++n) *reinterpret_cast<float2*>(to + n * 8) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
            }
        }
        w.next(a);
    }
    // ---- the warps' parts of an item: results where the block has all of them, else a part of the block.
    // A run of parts is one, and slot 0 of the warps behind up to one that ends the item.  Its rows are dealt out to the warps, eight columns to a thread, with
    // all parts asked for together: l = sum_i 2^(m_i - M) l_i and the like for o, in the order of the warps.
    // (Four parts at a time: one sequence of 16384 keys 16.2 us instead of 15.7, 9 x 4 tokens 22.4 instead of 21.8; four columns to a thread the same for these,
    // 64 ragged sequences 56.4 instead of 55.5.)
    __syncthreads();
    const int from = (lane >> 1) & (kFewWarps - 1), slot = lane & 1;
    int count = 0;
    bool ends = false;
    if (lane < 2 * kFewWarps && pieces[from][slot].rows > 0 && (slot || from == 0)) {      // (slot 0 of a later warp continues a run)
        count = 1;
        ends = pieces[from][slot].ends;
        while (!ends && from + count < kFewWarps && pieces[from + count][0].rows > 0) ends = pieces[from + count++][0].ends;
    }
    constexpr int LANES = D / 8, ROWS = 32 / LANES;               // threads of a row; rows of a warp at a time
    int turn = 0;
    for (uint32_t runs = __ballot_sync(0xffffffffu, count > 0); runs; runs &= runs - 1) {
        const int at = __ffs(runs) - 1, n = __shfl_sync(0xffffffffu, count, at), first = at >> 1, begins = at & 1;
        const bool done = __shfl_sync(0xffffffffu, ends, at) && begins;
        const Piece head = pieces[first][begins];
        const long long to = blockIdx.x * 2 + begins;
        if (begins && !done && threadIdx.x == 0)
            a.joins[blockIdx.x] = make_int4(head.last / kFewWarps - (int)blockIdx.x + 1, head.row0, head.rows, head.block);
        for (int r = 0; r < head.rows; r += ROWS, ++turn) {
            const int row = r + lane / LANES, col = lane % LANES * 8;
            if ((turn & (kFewWarps - 1)) != warp || row >= head.rows) continue;
            float2 st[kFewWarps];
            float4 v[kFewWarps][2], o[2] = {};
            float m = NEG_INF, l = 0.f;
            auto ask = [&](int k) {
                st[k] = make_float2(NEG_INF, 0.f);
                v[k][0] = v[k][1] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (k < n) {
                    const int w = first + k, sl = k ? 0 : begins;
                    st[k] = stats[w][sl][row];
                    const float* const src = pieces[w][sl].far ? own + (long long)(blockIdx.x * kFewWarps + w) * kFewRows * D
                                                               : reinterpret_cast<const float*>(smem + w * (kStagesFew * kUnitBytes));
                    v[k][0] = reinterpret_cast<const float4*>(src + row * D + col)[0];
                    v[k][1] = reinterpret_cast<const float4*>(src + row * D + col)[1];
                }
                m = fmaxf(m, st[k].x);
            };
            auto add = [&](int k) {
                if (st[k].x == NEG_INF) return;                  // (it saw no key)
                const float g = st[k].x == m ? 1.f : ex2(st[k].x - m);
                l += g * st[k].y;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    o[e].x += g * v[k][e].x; o[e].y += g * v[k][e].y; o[e].z += g * v[k][e].z; o[e].w += g * v[k][e].w;
                }
            };
            static_assert(kFewWarps == 8, "two halves of four");
#pragma unroll
            for (int k = 0; k < 4; ++k) ask(k);                  // all parts asked for together
            if (n > 4) {
#pragma unroll
                for (int k = 4; k < 8; ++k) ask(k);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) add(k);
            if (n > 4) {
#pragma unroll
                for (int k = 4; k < 8; ++k) add(k);
            }
            if (done) {
                write_result<DT, D>(a, head.row0, head.block, row, col, l, o[0], o[1]);
            } else {
                if (col == 0) a.stats[to * kFewRows + row] = make_float2(m, l);
                float4* const dst = reinterpret_cast<float4*>(a.part(to, D, row, col));
                dst[0] = o[0];
                dst[1] = o[1];
            }
        }
    }
}

template <int DT, int D, int HALVES>
cudaError_t launch(const AttnArgs& a, float* own, int blocks, cudaStream_t stream) {
    constexpr int bytes = kFewWarps * kStagesFew * kUnitBytes;
    static SharedMemory allowed;
    const cudaError_t e = allowed.allow((const void*)attend_few<DT, D, HALVES>, bytes);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute pdl;
    pdl.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kFewWarps * 32);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = stream;
    cfg.attrs = &pdl;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, attend_few<DT, D, HALVES>, a, own);
}

template <int DT, int D>
cudaError_t launch(const AttnArgs& a, float* own, int blocks, cudaStream_t stream) {
    return a.tokens * a.group <= 8 ? launch<DT, D, 1>(a, own, blocks, stream) : launch<DT, D, 2>(a, own, blocks, stream);
}

}  // namespace

cudaError_t launch_few(const AttnArgs& a, float* own, int head_dim, int dtype, int blocks, cudaStream_t stream) {
    if (dtype == DT_F16) return head_dim == 64 ? launch<DT_F16, 64>(a, own, blocks, stream) : launch<DT_F16, 128>(a, own, blocks, stream);
    return head_dim == 64 ? launch<DT_BF16, 64>(a, own, blocks, stream) : launch<DT_BF16, 128>(a, own, blocks, stream);
}

}  // namespace mk

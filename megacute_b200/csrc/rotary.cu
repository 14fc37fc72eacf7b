// Rotation of heads by their positions, by itself (mk_rotary) or on the way into a paged cache (mk_paged_append).
//
//   half:         y[i] = x[i] cos[p, i] - x[i + n] sin[p, i],  y[i + n] = x[i + n] cos[p, i] + x[i] sin[p, i]      i < n
//   interleaved:  the same for x[2 i], x[2 i + 1]
//
// in fp32, rounded once.  Bound by memory: every element is read and written once, a position's table row once per row.
// A thread's piece is 16 elements of a head (8 pairs: two 16-byte accesses of a 16-bit type, the same 8 table columns in both layouts) in up to four heads
// of a row (fp32: two), so that cosines and sines are fetched once for all of them; the next piece's elements are asked for before this one is turned.  A block has up
// to eight rows; its warps find the rows' sequences, positions and cache rows while the first elements come.
// Measured (5 prompts of up to 3271 rows, 32 heads of 128, 96 rotated; append of 4 x 4096 rows, 48 heads of 64): 23.5 and 40.5 us, 85 % and 77 % of the
// measured copy rate; blocks of 256 threads, one piece a thread, looked up first 26 and 49 us; two heads a piece 28.7 and 41.9.  fp32, 8192 rows of 32
// heads of 128: 47.8 us, 87 %, interleaved 51.7.
#include "paged.cuh"

namespace mk {
namespace {

constexpr int kRotThreads = 128;
constexpr int kRotRows = 8;                           // rows of a block, at most
constexpr int kRotBlocks = 148 * 4;                   // blocks that run at a time
template <int ES> constexpr int heads_of_thread = 8 / ES;

struct RotArgs {
    Batch batch;
    Pages pages;                                      // (append)
    const void* cos;
    const void* sin;
    const uint8_t* x;
    uint8_t* out;
    uint8_t* k;
    uint8_t* v;
    long long ld_cos, ld_sin, ld_x, ld_out, ld_k, ld_v;
    int tdtype, trows, columns;
    int heads, kv_heads, head_dim;
    int block_rows, groups;                           // rows of a block; threads that share a row's 16 elements of a head
};

template <int ES>
struct Sixteen {                                      // two vectors of 8 elements
    uint4 w[2][ES / 2];
};
template <int ES>
__device__ __forceinline__ void load16(Sixteen<ES>& s, const uint8_t* a, const uint8_t* b) {
#pragma unroll
    for (int i = 0; i < ES / 2; ++i) {
        s.w[0][i] = reinterpret_cast<const uint4*>(a)[i];
        s.w[1][i] = reinterpret_cast<const uint4*>(b)[i];
    }
}
template <int ES>
__device__ __forceinline__ void store16(const Sixteen<ES>& s, uint8_t* a, uint8_t* b) {
#pragma unroll
    for (int i = 0; i < ES / 2; ++i) {
        reinterpret_cast<uint4*>(a)[i] = s.w[0][i];
        reinterpret_cast<uint4*>(b)[i] = s.w[1][i];
    }
}
template <int DT>
__device__ __forceinline__ float2 get2(const uint4* w, int pair) {         // elements 2 pair, 2 pair + 1 of a vector
    const uint32_t* u = reinterpret_cast<const uint32_t*>(w);
    if (DT == DT_F32) return make_float2(__uint_as_float(u[2 * pair]), __uint_as_float(u[2 * pair + 1]));
    return unpack16<DT>(u[pair]);
}
template <int DT>
__device__ __forceinline__ void put2(uint4* w, int pair, float a, float b) {
    uint32_t* u = reinterpret_cast<uint32_t*>(w);
    if (DT == DT_F32) {
        u[2 * pair] = __float_as_uint(a);
        u[2 * pair + 1] = __float_as_uint(b);
    } else {
        u[pair] = pack16<DT>(a, b);
    }
}
__device__ __forceinline__ void table8(const void* t, int dtype, long long at, float* f) {
    if (dtype == DT_F32) {
        const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(t) + at);
        const float4 a = __ldg(p), b = __ldg(p + 1);
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
        return;
    }
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(t) + at));
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = dtype == DT_F16 ? unpack16<DT_F16>(u[i]) : unpack16<DT_BF16>(u[i]);
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
    }
}

enum { ROW_NONE = 0, ROW_ZERO = 1, ROW_TURN = 2 };

template <int DT, bool INTER, bool APPEND>
__global__ void __launch_bounds__(kRotThreads, 4) rotate_rows(const __grid_constant__ RotArgs a) {
    constexpr int ES = DT == DT_F32 ? 4 : 2, kHeads = heads_of_thread<ES>;
    __shared__ int s_state[kRotRows], s_pos[kRotRows], s_row[kRotRows];
    wait_for_previous_kernel();
    const int row0 = blockIdx.x * a.block_rows, rows = min(a.block_rows, a.batch.rows - row0);
    const int warp = threadIdx.x >> 5;
    const int slots = a.head_dim >> 4, heads = APPEND ? a.heads + 2 * a.kv_heads : a.heads;
    const int per_row = slots * a.groups, turned = APPEND ? a.heads + a.kv_heads : a.heads;
    // one of the rows' pieces: 16 elements of every groups-th head from `group` on
    struct Piece {
        int row, slot, group;
        Sixteen<ES> v[kHeads];
    };
    // the two vectors' first elements in a head
    auto place = [&](int slot, int& e0, int& e1) {
        const bool turn = slot < a.columns >> 3;
        e0 = turn && !INTER ? slot * 8 : slot * 16;
        e1 = turn && !INTER ? a.columns + slot * 8 : slot * 16 + 8;
        return turn;
    };
    auto request = [&](int u, Piece& w) {
        w.row = u / per_row;
        const int at = u - w.row * per_row;
        w.group = at / slots;
        w.slot = at - w.group * slots;
        int e0, e1;
        place(w.slot, e0, e1);
        const uint8_t* x = a.x + ((row0 + w.row) * a.ld_x + w.group * a.head_dim) * ES;
#pragma unroll
        for (int i = 0; i < kHeads; ++i, x += a.groups * a.head_dim * ES)
            if (w.group + i * a.groups < heads) load16(w.v[i], x + e0 * ES, x + e1 * ES);
    };
    int u = threadIdx.x;
    Piece w;
    if (u < rows * per_row) request(u, w);            // asked for before it is known where it goes
    for (int i = warp; i < rows; i += kRotThreads / 32) {
        const int r = row0 + i, s = sequence_of_row(a.batch, r);
        int state = ROW_NONE, cache_row = -1;
        long long p = 0;
        if (s >= 0) {
            p = (long long)a.batch.position(s) + (r - a.batch.first(s));
            state = p >= 0 && p < a.trows ? ROW_TURN : ROW_ZERO;
            if (APPEND) {
                if (p >= a.pages.capacity()) state = ROW_ZERO;
                if (state == ROW_TURN) {
                    const int first = a.pages.page_row(s, (int)p >> a.pages.shift);
                    if (first >= 0) cache_row = first + ((int)p & ((1 << a.pages.shift) - 1));
                }
            }
        }
        if ((threadIdx.x & 31) == 0) {
            s_state[i] = state;
            s_pos[i] = (int)p;
            s_row[i] = cache_row;
        }
    }
    __syncthreads();
    auto turn_piece = [&](Piece& w) {
        const int state = s_state[w.row];
        if (state == ROW_NONE) return;
        const long long r = row0 + w.row;
        int e0, e1;
        const bool turn = place(w.slot, e0, e1);
        float c[8], s[8];
        if (turn && state == ROW_TURN) {
            table8(a.cos, a.tdtype, s_pos[w.row] * a.ld_cos + w.slot * 8, c);
            table8(a.sin, a.tdtype, s_pos[w.row] * a.ld_sin + w.slot * 8, s);
        }
        const long long cache_row = s_row[w.row];
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            const int h = w.group + i * a.groups;
            if (h >= heads) break;
            if (state == ROW_ZERO) {
#pragma unroll
                for (int e = 0; e < ES / 2; ++e) w.v[i].w[0][e] = w.v[i].w[1][e] = make_uint4(0, 0, 0, 0);
            } else if (turn && h < turned) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (INTER) {                                           // pairs 2 e, 2 e + 1: words of one vector
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const int j = 2 * e + k;
                            const float2 z = get2<DT>(w.v[i].w[j >> 2], j & 3);
                            put2<DT>(w.v[i].w[j >> 2], j & 3, z.x * c[j] - z.y * s[j], z.y * c[j] + z.x * s[j]);
                        }
                    } else {
                        const float2 lo = get2<DT>(w.v[i].w[0], e), hi = get2<DT>(w.v[i].w[1], e);
                        put2<DT>(w.v[i].w[0], e, lo.x * c[2 * e] - hi.x * s[2 * e], lo.y * c[2 * e + 1] - hi.y * s[2 * e + 1]);
                        put2<DT>(w.v[i].w[1], e, hi.x * c[2 * e] + lo.x * s[2 * e], hi.y * c[2 * e + 1] + lo.y * s[2 * e + 1]);
                    }
                }
            }
            uint8_t* to;
            if (!APPEND || h < a.heads) {
                to = a.out + (r * a.ld_out + h * a.head_dim) * ES;
            } else {
                if (cache_row < 0) continue;
                to = h < turned ? a.k + (cache_row * a.ld_k + (h - a.heads) * a.head_dim) * ES
                                : a.v + (cache_row * a.ld_v + (h - turned) * a.head_dim) * ES;
            }
            store16(w.v[i], to + e0 * ES, to + e1 * ES);
        }
    };
    while (u < rows * per_row) {
        Piece next;
        u += kRotThreads;
        if (u < rows * per_row) request(u, next);     // (under way while this one is turned)
        turn_piece(w);
        w = next;
    }
}
int launch(RotArgs& a, int dtype, bool inter, bool append, void* stream) {
    const int heads = append ? a.heads + 2 * a.kv_heads : a.heads, slots = a.head_dim >> 4;
    const int each = dtype == DT_F32 ? heads_of_thread<4> : heads_of_thread<2>;
    a.groups = (heads + each - 1) / each;
    const int per_row = slots * a.groups;
    // rows of a block: at least as many as give each thread a piece, else so many that the blocks fill whole rounds of the SMs (a block begins with a chain of
    // look-ups, so few rounds; 4 x 4096 rows in 3.5 rounds of 8 rows 41.4 us, in 4 of 7 40.4, in 2 of 14 40.2; 5 prompts 24.7, 23.5 and 30)
    const int least = max(1, kRotThreads / per_row), rounds = (a.batch.rows - 1) / (kRotBlocks * kRotRows) + 1;
    a.block_rows = min(kRotRows, max(least, (a.batch.rows - 1) / (kRotBlocks * rounds) + 1));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((a.batch.rows + a.block_rows - 1) / a.block_rows));
    cfg.blockDim = dim3(kRotThreads);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute pdl;
    pdl.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &pdl;
    cfg.numAttrs = 1;
    cudaError_t e;
#define MK_ROT(DT, APPEND) e = inter ? cudaLaunchKernelEx(&cfg, rotate_rows<DT, true, APPEND>, a) : cudaLaunchKernelEx(&cfg, rotate_rows<DT, false, APPEND>, a)
    if (append) {
        if (dtype == DT_BF16) MK_ROT(DT_BF16, true);
        else MK_ROT(DT_F16, true);
    } else {
        if (dtype == DT_BF16) MK_ROT(DT_BF16, false);
        else if (dtype == DT_F16) MK_ROT(DT_F16, false);
        else MK_ROT(DT_F32, false);
    }
#undef MK_ROT
    if (e == cudaSuccess) return MK_OK;
    (void)cudaGetLastError();
    return report(MK_E_CUDA, cudaGetErrorString(e));
}

RotArgs args_of(const mk_batch* b, const mk_rotation* r) {
    RotArgs a = {};
    a.batch = batch_of(b);
    a.cos = r->cos;
    a.sin = r->sin;
    a.ld_cos = r->ld_cos;
    a.ld_sin = r->ld_sin;
    a.tdtype = r->dtype;
    a.trows = r->rows;
    a.columns = r->columns;
    return a;
}

}  // namespace
}  // namespace mk

using namespace mk;

extern "C" int mk_rotary(int device, const mk_batch* batch, const mk_rotation* rot, const void* x, int64_t ld_x, void* out, int64_t ld_out,
                         int dtype, int heads, int head_dim, void* stream) {
    const char* why = batch_error(batch);
    if (!why && (heads <= 0 || head_dim <= 0 || head_dim % 16)) why = "rotary: head_dim is a multiple of 16";
    if (!why) why = rotation_error(rot, head_dim);
    if (!why && (dtype < DT_BF16 || dtype > DT_F16)) why = "rotary: bf16, fp32 or fp16";
    if (why) return report(MK_E_ARG, why);
    if (batch->rows == 0 || batch->seqs == 0) return MK_OK;
    const long long width = (long long)heads * head_dim;
    const int es = elem_bytes(dtype);
    if (!x || !out || width > 0x1fffffff || ld_x < width || ld_out < width || !aligned16(x, ld_x, es) || !aligned16(out, ld_out, es))
        return report(MK_E_ARG, "rotary: rows hold all heads and start on 16-byte boundaries");
    OnDevice on(device);
    if (!on.ok) return report(MK_E_CUDA, "cudaSetDevice");
    RotArgs a = args_of(batch, rot);
    a.x = (const uint8_t*)x;
    a.out = (uint8_t*)out;
    a.ld_x = ld_x;
    a.ld_out = ld_out;
    a.heads = heads;
    a.head_dim = head_dim;
    return launch(a, dtype, rot->interleaved != 0, false, stream);
}

extern "C" int mk_paged_append(int device, const mk_batch* batch, const mk_rotation* rot, const mk_paged_cache* cache, const void* qkv,
                               int64_t ld_qkv, void* q_out, int64_t ld_q, int heads, void* stream) {
    const char* why = batch_error(batch);
    if (!why) why = cache_error(cache);
    if (!why && (heads <= 0 || cache->head_dim % 16)) why = "paged append: head_dim is a multiple of 16";
    if (!why) why = rotation_error(rot, cache->head_dim);
    if (why) return report(MK_E_ARG, why);
    if (batch->rows == 0 || batch->seqs == 0) return MK_OK;
    const long long width = ((long long)heads + 2ll * cache->kv_heads) * cache->head_dim, q_width = (long long)heads * cache->head_dim;
    if (!qkv || !q_out || width > 0x1fffffff || ld_qkv < width || ld_q < q_width || !aligned16(qkv, ld_qkv, 2) || !aligned16(q_out, ld_q, 2))
        return report(MK_E_ARG, "paged append: rows hold all heads and start on 16-byte boundaries");
    OnDevice on(device);
    if (!on.ok) return report(MK_E_CUDA, "cudaSetDevice");
    RotArgs a = args_of(batch, rot);
    a.pages = pages_of(cache);
    a.x = (const uint8_t*)qkv;
    a.out = (uint8_t*)q_out;
    a.k = (uint8_t*)cache->k;
    a.v = (uint8_t*)cache->v;
    a.ld_x = ld_qkv;
    a.ld_out = ld_q;
    a.ld_k = cache->ld_k;
    a.ld_v = cache->ld_v;
    a.heads = heads;
    a.kv_heads = cache->kv_heads;
    a.head_dim = cache->head_dim;
    return launch(a, cache->dtype, rot->interleaved != 0, true, stream);
}

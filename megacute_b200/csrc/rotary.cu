// Rotation of heads by their positions, by itself (mk_rotary) or on the way into a paged cache (mk_paged_append).
//
//   half:         y[i] = x[i] cos[p, i] - x[i + n] sin[p, i],  y[i + n] = x[i + n] cos[p, i] + x[i] sin[p, i]      i < n
//   interleaved:  the same for x[2 i], x[2 i + 1]
//
// in fp32, rounded once.  Bound by memory: every element is read and written once, a position's table row once per row.
// A thread owns 16 elements of a head (8 pairs: two 16-byte accesses of a 16-bit type, the same 8 table columns in both layouts) and
// takes them through up to kHeads heads of the row, so that its cosines and sines are fetched once and its loads of all those heads are
// under way together.  A block has up to eight rows; one warp per row finds the row's sequence, position and cache row while the elements come.
#include "paged.cuh"

namespace mk {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotRows = kRotThreads / 32;            // rows of a block, at most
constexpr int kHeads = 4;

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
__global__ void __launch_bounds__(kRotThreads) rotate_rows(const __grid_constant__ RotArgs a) {
    constexpr int ES = DT == DT_F32 ? 4 : 2;
    __shared__ int s_state[kRotRows], s_pos[kRotRows], s_row[kRotRows];
    wait_for_previous_kernel();
    const int row0 = blockIdx.x * a.block_rows, rows = min(a.block_rows, a.batch.rows - row0);
    const int warp = threadIdx.x >> 5;
    const int slots = a.head_dim >> 4, heads = APPEND ? a.heads + 2 * a.kv_heads : a.heads;
    const int per_row = slots * a.groups, turned = APPEND ? a.heads + a.kv_heads : a.heads;
    // what thread u of the rows' does: a row, 16 elements of a head, every groups-th head from `group` on
    int u = threadIdx.x, row, slot, group, e0, e1;
    bool turn;
    Sixteen<ES> v[kHeads];
    auto request = [&] {                              // its elements: asked for before it is known where they go
        row = u / per_row;
        const int at = u - row * per_row;
        slot = at % slots;
        group = at / slots;
        turn = slot < a.columns >> 3;
        // the two vectors' first elements in a head
        e0 = turn && !INTER ? slot * 8 : slot * 16;
        e1 = turn && !INTER ? a.columns + slot * 8 : slot * 16 + 8;
        const uint8_t* x = a.x + (row0 + row) * a.ld_x * ES;
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            const int h = group + i * a.groups;
            if (h < heads) load16(v[i], x + (h * a.head_dim + e0) * ES, x + (h * a.head_dim + e1) * ES);
        }
    };
    if (u < rows * per_row) request();
    if (warp < rows) {
        const int r = row0 + warp, s = sequence_of_row(a.batch, r);
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
            s_state[warp] = state;
            s_pos[warp] = (int)p;
            s_row[warp] = cache_row;
        }
    }
    __syncthreads();
    for (; u < rows * per_row; u += kRotThreads) {
        if (u >= kRotThreads) request();
        const int state = s_state[row];
        if (state == ROW_NONE) continue;
        const long long r = row0 + row;
        float c[8], s[8];
        if (turn && state == ROW_TURN) {
            table8(a.cos, a.tdtype, s_pos[row] * a.ld_cos + slot * 8, c);
            table8(a.sin, a.tdtype, s_pos[row] * a.ld_sin + slot * 8, s);
        }
        const long long cache_row = s_row[row];
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            const int h = group + i * a.groups;
            if (h >= heads) break;
            if (state == ROW_ZERO) {
#pragma unroll
                for (int e = 0; e < ES / 2; ++e) v[i].w[0][e] = v[i].w[1][e] = make_uint4(0, 0, 0, 0);
            } else if (turn && h < turned) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (INTER) {                                           // pairs 2 e, 2 e + 1: words of one vector
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const int j = 2 * e + k;
                            const float2 z = get2<DT>(v[i].w[j >> 2], j & 3);
                            put2<DT>(v[i].w[j >> 2], j & 3, z.x * c[j] - z.y * s[j], z.y * c[j] + z.x * s[j]);
                        }
                    } else {
                        const float2 lo = get2<DT>(v[i].w[0], e), hi = get2<DT>(v[i].w[1], e);
                        put2<DT>(v[i].w[0], e, lo.x * c[2 * e] - hi.x * s[2 * e], lo.y * c[2 * e + 1] - hi.y * s[2 * e + 1]);
                        put2<DT>(v[i].w[1], e, hi.x * c[2 * e] + lo.x * s[2 * e], hi.y * c[2 * e + 1] + lo.y * s[2 * e + 1]);
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
            store16(v[i], to + e0 * ES, to + e1 * ES);
        }
    }
}

int launch(RotArgs& a, int dtype, bool inter, bool append, void* stream) {
    const int heads = append ? a.heads + 2 * a.kv_heads : a.heads, slots = a.head_dim >> 4;
    a.groups = (heads + kHeads - 1) / kHeads;
    const int per_row = slots * a.groups;
    a.block_rows = min(kRotRows, max(1, kRotThreads / per_row));
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
    if (!x || !out || width > 0x3fffffff || ld_x < width || ld_out < width || !aligned16(x, ld_x, es) || !aligned16(out, ld_out, es))
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
    if (!qkv || !q_out || width > 0x3fffffff || ld_qkv < width || ld_q < q_width || !aligned16(qkv, ld_qkv, 2) || !aligned16(q_out, ld_q, 2))
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

// Attention of new tokens over a paged cache (mk_paged_attention): the entry points, the choice of kernel, and the kernel that joins
// the parts of items that several workers had.
//
//   out[r, h] = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   s_j = scale q[r, h] . k_j,   j in [max(0, p + 1 - window), p]
#include "paged_attention.cuh"

namespace mk {
namespace {

constexpr int kJoinThreads = 256;
constexpr int kJoinRows = 16;                         // rows of a block

// Block (x, y): items that the workers [x * per_block, (x + 1) * per_block) begin and do not end, rows [y * kJoinRows, ...) of them.
// With M the largest of the parts' maxima m_i: out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i, in the order of the parts.
// A warp has a row; where there are fewer rows than warps, several warps share a row's parts and add through shared memory.
template <int DT, int D>
__global__ void __launch_bounds__(kJoinThreads) join_parts(const __grid_constant__ AttnArgs a, int per_block) {
    constexpr int V = D / 32, WARPS = kJoinThreads / 32;
    __shared__ float sums[WARPS][D];
    wait_for_previous_kernel();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int w = blockIdx.x * per_block; w < (blockIdx.x + 1) * per_block; ++w) {
        const int4 j = __ldcg(a.joins + w);
        const int first = blockIdx.y * kJoinRows, rows = min(kJoinRows, j.z - first);
        if (j.x == 0 || rows <= 0) continue;
        int across = 1;                               // rows side by side
        while (across < rows && across < WARPS) across <<= 1;
        const int split = warp / across, splits = WARPS / across;
        for (int r = warp % across; r < (rows + across - 1) / across * across; r += across) {
            const int row = first + min(r, rows - 1);
            auto slot = [&](int i) { return (long long)(i == 0 ? 2 * w + 1 : 2 * (w + i)) * a.part_rows + row; };
            float m = -__builtin_huge_valf(), l = 0.f;
            for (int i = lane; i < j.x; i += 32) {
                const float2 st = __ldcg(reinterpret_cast<const float2*>(a.stats) + slot(i));
                const float to = fmaxf(m, st.x);
                if (to != -__builtin_huge_valf()) l = l * (m == to ? 1.f : ex2(m - to)) + st.y * (st.x == to ? 1.f : ex2(st.x - to));
                m = to;
            }
#pragma unroll
            for (int d = 16; d; d >>= 1) {
                const float m2 = __shfl_xor_sync(0xffffffffu, m, d), l2 = __shfl_xor_sync(0xffffffffu, l, d), to = fmaxf(m, m2);
                if (to != -__builtin_huge_valf()) l = l * (m == to ? 1.f : ex2(m - to)) + l2 * (m2 == to ? 1.f : ex2(m2 - to));
                m = to;
            }
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = 0.f;
            if (m != -__builtin_huge_valf()) {
#pragma unroll 4
                for (int i = split; i < j.x; i += splits) {
                    const long long at = slot(i);
                    const float mi = __ldcg(a.stats + 2 * at), f = mi == m ? 1.f : ex2(mi - m);
                    float x[V];
                    if (V == 4) {
                        const float4 t = __ldcg(reinterpret_cast<const float4*>(a.parts + at * D) + lane);
                        x[0] = t.x; x[1] = t.y; x[V - 2] = t.z; x[V - 1] = t.w;
                    } else {
                        const float2 t = __ldcg(reinterpret_cast<const float2*>(a.parts + at * D) + lane);
                        x[0] = t.x; x[1] = t.y;
                    }
                    if (mi != -__builtin_huge_valf()) {
#pragma unroll
                        for (int e = 0; e < V; ++e) o[e] += f * x[e];
                    }
                }
            }
            if (splits > 1) {                         // (one turn of the loop over rows: across >= rows)
                __syncthreads();
#pragma unroll
                for (int e = 0; e < V; ++e) sums[warp][lane * V + e] = o[e];
                __syncthreads();
                if (split > 0) continue;
                for (int k = 1; k < splits; ++k)
#pragma unroll
                    for (int e = 0; e < V; ++e) o[e] += sums[warp + k * across][lane * V + e];
            }
            if (r >= rows) continue;
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const int tok = row / a.group;
            uint32_t* to = reinterpret_cast<uint32_t*>(a.out + (j.y + tok) * a.ld_out + (j.w * a.group + row - tok * a.group) * D) + lane * (V / 2);
            if (V == 4) *reinterpret_cast<uint2*>(to) = make_uint2(pack16<DT>(o[0] * inv, o[1] * inv), pack16<DT>(o[V - 2] * inv, o[V - 1] * inv));
            else *to = pack16<DT>(o[0] * inv, o[1] * inv);
        }
    }
}

const char* shape_error(const mk_paged_cache* cache, int heads) {
    const char* why = cache_error(cache);
    if (!why && cache->head_dim != 64 && cache->head_dim != 128) why = "paged attention: head_dim is 64 or 128";
    if (!why && (heads <= 0 || heads % cache->kv_heads)) why = "paged attention: heads is a multiple of kv_heads";
    return why;
}

int sm_count(int device) {
    static int counts[64] = {};
    if (device < 0 || device >= 64) return 0;
    if (counts[device] == 0) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
            (void)cudaGetLastError();
            return 0;
        }
        counts[device] = n;
    }
    return counts[device];
}

// heads of an item of at most `rows` rows: those of a kv head, or a divisor of their number
int heads_of_block(int group, int rows) {
    int n = group;
    for (int parts = 2; n > rows; ++parts)
        if (group % parts == 0) n = group / parts;
    return n;
}

// Which kernel takes a call: the one for few rows where an item of 16 rows holds all new tokens of a sequence (then every key is read once).
bool few_rows(int group, long long max_new) { return max_new * group <= kFewRows; }

// what the workspace holds, one behind the other: joins, stats, parts
struct Layout {
    int workers, part_rows, per_block;
    size_t stats, parts, bytes;
};
Layout layout_of(int sms, int head_dim, bool few) {
    Layout l;
    l.per_block = few ? kFewWarps : 1;
    l.workers = sms * l.per_block;
    l.part_rows = few ? kFewRows : 2 * kChunkTile;
    l.stats = (size_t)l.workers * sizeof(int4);
    l.parts = l.stats + (size_t)l.workers * 2 * l.part_rows * 2 * sizeof(float);
    l.bytes = l.parts + (size_t)l.workers * 2 * l.part_rows * head_dim * sizeof(float);
    return l;
}

template <int DT, int D>
cudaError_t launch_join(const AttnArgs& a, int per_block, cudaStream_t stream) {
    cudaLaunchAttribute pdl;
    pdl.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.workers / per_block), (unsigned)((a.part_rows + kJoinRows - 1) / kJoinRows));
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = stream;
    cfg.attrs = &pdl;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, join_parts<DT, D>, a, per_block);
}

}  // namespace
}  // namespace mk

using namespace mk;

extern "C" long long mk_paged_attention_workspace(int device, int heads, const mk_paged_cache* cache, int max_new) {
    const char* why = shape_error(cache, heads);
    if (why) return report(MK_E_ARG, why);
    const int sms = sm_count(device);
    if (!sms) return report(MK_E_CUDA, "no such device");
    const size_t few = layout_of(sms, cache->head_dim, true).bytes, chunk = layout_of(sms, cache->head_dim, false).bytes;
    // (a scale that is not positive is for the kernel for few rows, whatever max_new)
    return (long long)(few_rows(heads / cache->kv_heads, max_new) || few > chunk ? few : chunk);
}

extern "C" int mk_paged_attention(int device, const mk_batch* batch, const mk_paged_cache* cache, const void* q, int64_t ld_q, void* out,
                                  int64_t ld_out, int heads, float scale, int window, int max_new, void* workspace, size_t workspace_bytes,
                                  void* stream) {
    const char* why = batch_error(batch);
    if (!why) why = shape_error(cache, heads);
    if (!why && window < 0) why = "paged attention: window is a number of rows (0: the whole context)";
    if (why) return report(MK_E_ARG, why);
    if (batch->rows == 0 || batch->seqs == 0) return MK_OK;
    const int D = cache->head_dim, group = heads / cache->kv_heads;
    const long long width = (long long)heads * D;
    if (!q || !out || ld_q < width || ld_out < width || !aligned16(q, ld_q, 2) || !aligned16(out, ld_out, 2))
        return report(MK_E_ARG, "paged attention: rows hold all heads and start on 16-byte boundaries");
    if (!workspace || ((uintptr_t)workspace & 15)) return report(MK_E_ARG, "paged attention: workspace of 16-byte aligned device memory");
    const int sms = sm_count(device);
    if (!sms) return report(MK_E_CUDA, "no such device");
    const bool few = few_rows(group, max_new) || !(scale > 0.f) || scale > 1e30f;
    const Layout lay = layout_of(sms, D, few);
    if (workspace_bytes < lay.bytes) return report(MK_E_ARG, "paged attention: workspace smaller than mk_paged_attention_workspace()");
    OnDevice on(device);
    if (!on.ok) return report(MK_E_CUDA, "cudaSetDevice");
    AttnArgs a = {};
    a.batch = batch_of(batch);
    a.pages = pages_of(cache);
    a.q = (const uint16_t*)q;
    a.k = (const uint16_t*)cache->k;
    a.v = (const uint16_t*)cache->v;
    a.out = (uint16_t*)out;
    a.ld_q = ld_q;
    a.ld_k = cache->ld_k;
    a.ld_v = cache->ld_v;
    a.ld_out = ld_out;
    a.group = heads_of_block(group, few ? kFewRows : kChunkTile);
    a.shared = group / a.group;
    a.blocks = heads / a.group;
    a.window = window;
    a.scale2 = scale * kLog2e;
    a.workers = lay.workers;
    a.part_rows = lay.part_rows;
    a.joins = (int4*)workspace;
    a.stats = (float*)((uint8_t*)workspace + lay.stats);
    a.parts = (float*)((uint8_t*)workspace + lay.parts);
    cudaStream_t st = (cudaStream_t)stream;
    a.tokens = few ? kFewRows / a.group : kChunkTile / a.group * 2;
    cudaError_t e = few ? launch_few(a, D, cache->dtype, sms, st) : launch_chunk(a, cache, heads, st);
    if (e == cudaSuccess) {
        if (cache->dtype == DT_F16) e = D == 64 ? launch_join<DT_F16, 64>(a, lay.per_block, st) : launch_join<DT_F16, 128>(a, lay.per_block, st);
        else e = D == 64 ? launch_join<DT_BF16, 64>(a, lay.per_block, st) : launch_join<DT_BF16, 128>(a, lay.per_block, st);
    }
    if (e == cudaSuccess) return MK_OK;
    (void)cudaGetLastError();
    return report(MK_E_CUDA, cudaGetErrorString(e));
}

extern "C" int mk_paged_attention_status(int device, void* stream) {
    OnDevice on(device);
    if (!on.ok) return report(MK_E_CUDA, "cudaSetDevice");
    int failed = 0;
    const cudaError_t e = chunk_status(&failed, (cudaStream_t)stream);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return report(MK_E_CUDA, cudaGetErrorString(e));
    }
    return failed ? MK_E_DEVICE : MK_OK;
}

// Attention of new tokens over a paged cache (mk_paged_attention): the entry points, the choice of kernel, and the kernel that joins
// the parts of items that several workers had.
//
//   out[r, h] = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   s_j = scale q[r, h] . k_j,   j in [max(0, p + 1 - window), p]
#include "paged_attention.cuh"

namespace mk {
namespace {

constexpr int kJoinThreads = 256;

// Block (x, y): the item that block x begins and does not end, rows [y * ROWS, (y + 1) * ROWS) of it.  Bound by latency: three dependent reads (the item, the
// statistics and products together, the next two parts) between the end of the kernel in front and its own, 3 to 5 us in all; its blocks are there
// before that kernel ends.  A grid of only the items that need it, found in front of the join, took longer than blocks that find nothing and leave.
template <int DT, int D, int ROWS>
__global__ void __launch_bounds__(kJoinThreads) join_parts(const __grid_constant__ AttnArgs a) {
    __shared__ Join<D, ROWS, kJoinThreads> join;
    wait_for_previous_kernel();
    const int w = blockIdx.x, first = blockIdx.y * ROWS;
    const int4 j = __ldcg(a.joins + w);
    if (j.x == 0 || first >= j.z) return;
    join.run(a, j.x, first, min(first + ROWS, j.z), [&](int i) { return (long long)(i == 0 ? 2 * w + 1 : 2 * (w + i)); },
             [&](int row, int col, float l, const float4& x, const float4& y) {
                 write_result<DT, D>(a, j.y, j.w, row, col, l, x, y);
             });
}

const char* shape_error(int heads, int kv_heads, int head_dim) {
    if (head_dim != 64 && head_dim != 128) return "paged attention: head_dim is 64 or 128";
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads) return "paged attention: heads is a multiple of kv_heads";
    return nullptr;
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
// Few rows and chunk kernel in us, 16 sequences of 4000 keys, bf16, group x tokens: 4 kv heads of 128, 4 x 2 33 and 37, 4 x 4 35 and 38, 4 x 5 60 and 38 (keys
// read twice); 8 kv heads of 64, 8 x 1 32 and 45, 8 x 2 34 and 45; 12 kv heads of 128, 1 x 16 78 and 86.
bool few_rows(int group, long long max_new) { return max_new * group <= kFewRows; }
// The hint as both entries take it: an item has a token at least.
int tokens_hinted(int max_new) { return max(max_new, 1); }

// what the workspace holds, one behind the other: joins, stats and parts of the blocks, parts of the warps (few rows)
struct Layout {
    int workers, part_rows;
    size_t stats, parts, own, bytes;
};
Layout layout_of(int sms, int head_dim, bool few) {
    Layout l;
    l.workers = few ? sms * kFewWarps : sms;
    l.part_rows = few ? kFewRows : 2 * kChunkTile;
    const size_t rows = (size_t)sms * 2 * l.part_rows;
    l.stats = ((size_t)sms * sizeof(int4) + 255) / 256 * 256;
    l.parts = l.stats + rows * sizeof(float2);
    l.own = l.parts + rows * head_dim * sizeof(float);
    l.bytes = l.own + (few ? (size_t)l.workers * kFewRows * head_dim * sizeof(float) : 0);
    return l;
}

template <int DT, int D, int ROWS>
cudaError_t launch_join(const AttnArgs& a, int blocks, cudaStream_t stream) {
    cudaLaunchAttribute pdl;
    pdl.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks, (unsigned)((a.tokens * a.group + ROWS - 1) / ROWS));
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = stream;
    cfg.attrs = &pdl;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, join_parts<DT, D, ROWS>, a);
}

}  // namespace
}  // namespace mk

using namespace mk;

extern "C" long long mk_paged_attention_workspace(int device, int heads, int kv_heads, int head_dim, int max_new) {
    const char* why = shape_error(heads, kv_heads, head_dim);
    if (why) return report(MK_E_ARG, why);
    const int sms = sm_count(device);
    if (!sms) return report(MK_E_CUDA, "no such device");
    const size_t few = layout_of(sms, head_dim, true).bytes, chunk = layout_of(sms, head_dim, false).bytes;
    // (a scale that is not positive is for the kernel for few rows, whatever max_new)
    return (long long)(few_rows(heads / kv_heads, tokens_hinted(max_new)) || few > chunk ? few : chunk);
}

extern "C" int mk_paged_attention(int device, const mk_batch* batch, const mk_paged_cache* cache, const void* q, int64_t ld_q, void* out,
                                  int64_t ld_out, int heads, float scale, int window, int max_new, void* workspace, size_t workspace_bytes,
                                  void* stream) {
    const char* why = batch_error(batch);
    if (!why) why = cache_error(cache);
    if (!why) why = shape_error(heads, cache->kv_heads, cache->head_dim);
    if (!why && window < 0) why = "paged attention: window is a number of rows (0: the whole context)";
    if (why) return report(MK_E_ARG, why);
    if (batch->rows == 0 || batch->seqs == 0) return MK_OK;
    max_new = tokens_hinted(max_new);
    const int D = cache->head_dim, group = heads / cache->kv_heads;
    const long long width = (long long)heads * D;
    if (!q || !out || ld_q < width || ld_out < width || !aligned16(q, ld_q, 2) || !aligned16(out, ld_out, 2))
        return report(MK_E_ARG, "paged attention: rows hold all heads and start on 16-byte boundaries");
    if (!workspace || ((uintptr_t)workspace & 255)) return report(MK_E_ARG, "paged attention: workspace of 256-byte aligned device memory");
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
    // (without pages no row is read; the addresses are ones of this call all the same)
    a.k = (const uint16_t*)(cache->pages ? cache->k : q);
    a.v = (const uint16_t*)(cache->pages ? cache->v : q);
    a.out = (uint16_t*)out;
    a.ld_q = ld_q;
    a.ld_k = cache->ld_k;
    a.ld_v = cache->ld_v;
    a.ld_out = ld_out;
    a.group = heads_of_block(group, few ? kFewRows : kChunkTile);
    a.group_inverse = 65536 / a.group + 1;
    a.shared = group / a.group;
    a.blocks = heads / a.group;
    a.window = window;
    a.scale2 = scale * kLog2e;
    a.workers = lay.workers;
    a.part_rows = lay.part_rows;
    a.joins = (int4*)workspace;
    a.stats = (float2*)((uint8_t*)workspace + lay.stats);
    a.parts = (float*)((uint8_t*)workspace + lay.parts);
    cudaStream_t st = (cudaStream_t)stream;
    // (8 rows an item where these hold all new tokens: half of the matrix instruction's rows, and nothing is done for the others)
    const int few_rows_of = (long long)max_new * a.group <= kFewRows / 2 ? kFewRows / 2 : kFewRows;
    a.tokens = few ? few_rows_of / a.group : kChunkTile / a.group * 2;
    a.align = few ? 16 : cache->page_size < kChunkTile ? cache->page_size : kChunkTile;
    float* const own = (float*)((uint8_t*)workspace + lay.own);
    cudaError_t e = few ? launch_few(a, own, D, cache->dtype, sms, st) : launch_chunk(a, cache, heads, st);
    if (e == cudaSuccess) {
        // (few rows of many parts, which several threads share; or many rows of few, with all parts in one thread: 16 rows of 64 columns, in two
        // threads each, took 4 x 4096 tokens 398.4 us instead of 396.6)
        if (few && cache->dtype == DT_F16) e = D == 64 ? launch_join<DT_F16, 64, 4>(a, sms, st) : launch_join<DT_F16, 128, 4>(a, sms, st);
        else if (few) e = D == 64 ? launch_join<DT_BF16, 64, 4>(a, sms, st) : launch_join<DT_BF16, 128, 4>(a, sms, st);
        else if (cache->dtype == DT_F16) e = D == 64 ? launch_join<DT_F16, 64, 32>(a, sms, st) : launch_join<DT_F16, 128, 16>(a, sms, st);
        else e = D == 64 ? launch_join<DT_BF16, 64, 32>(a, sms, st) : launch_join<DT_BF16, 128, 16>(a, sms, st);
    }
    if (e == cudaSuccess) return MK_OK;
    (void)cudaGetLastError();
    return report(MK_E_CUDA, cudaGetErrorString(e));
}

extern "C" int mk_paged_attention_failures(int device, void* stream, uint32_t* count) {
    if (!count) return report(MK_E_ARG, "paged attention: no place for the count");
    OnDevice on(device);
    if (!on.ok) return report(MK_E_CUDA, "cudaSetDevice");
    unsigned failed = 0;
    const cudaError_t e = chunk_failures(&failed, (cudaStream_t)stream);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return report(MK_E_CUDA, cudaGetErrorString(e));
    }
    *count = failed;
    return MK_OK;
}

extern "C" int mk_paged_attention_status(int device, void* stream) {
    uint32_t failed = 0;
    const int rc = mk_paged_attention_failures(device, stream, &failed);
    return rc != MK_OK ? rc : failed ? MK_E_DEVICE : MK_OK;
}

// Attention of new tokens over a paged cache (mk_paged_attention).
//
//   out[r, h] = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   s_j = scale q[r, h] . k_j,   j in [max(0, p + 1 - window), p]
//
// One warp per (row, head): a running maximum and sum over the row's keys one by one, the head's elements spread over the lanes.
#include "paged.cuh"

namespace mk {
namespace {

struct AttnArgs {
    Batch batch;
    Pages pages;
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* out;
    long long ld_q, ld_k, ld_v, ld_out;
    int heads, group, window;
    float scale2;                                     // scale * log2(e)
};

template <int DT, int D>
__global__ void __launch_bounds__(128) attend_row(const __grid_constant__ AttnArgs a) {
    constexpr int N = D / 64;                         // words of a lane
    const int lane = threadIdx.x & 31;
    const long long r = blockIdx.x;
    const int h = blockIdx.y * 4 + (threadIdx.x >> 5);
    if (h >= a.heads) return;
    const int s = sequence_of_row(a.batch, (int)r);
    if (s < 0) return;
    const long long p = (long long)a.batch.position(s) + (r - a.batch.first(s));
    const int hi = (int)min(p, (long long)a.pages.capacity() - 1);
    const int lo = a.window > 0 ? (int)min(max(p + 1 - a.window, 0ll), (long long)a.pages.capacity()) : 0;
    float2 q[N], o[N];
    for (int i = 0; i < N; ++i) {
        q[i] = unpack16<DT>(reinterpret_cast<const uint32_t*>(a.q + r * a.ld_q + h * D)[lane + 32 * i]);
        o[i] = make_float2(0.f, 0.f);
    }
    float m = -__builtin_huge_valf(), l = 0.f;
    bool any = false;
    const int kv = h / a.group;
    for (int j = lo; j <= hi; ++j) {
        const int first = a.pages.page_row(s, j >> a.pages.shift);
        if (first < 0) {
            j |= (1 << a.pages.shift) - 1;
            continue;
        }
        const long long row = first + (j & ((1 << a.pages.shift) - 1));
        float dot = 0.f;
        for (int i = 0; i < N; ++i) {
            const float2 k = unpack16<DT>(reinterpret_cast<const uint32_t*>(a.k + row * a.ld_k + kv * D)[lane + 32 * i]);
            dot += q[i].x * k.x + q[i].y * k.y;
        }
        for (int d = 16; d; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
        const float t = dot * a.scale2, mn = any ? fmaxf(m, t) : t, f = any ? exp2f(m - mn) : 0.f, e = exp2f(t - mn);
        any = true;
        l = l * f + e;
        m = mn;
        for (int i = 0; i < N; ++i) {
            const float2 v = unpack16<DT>(reinterpret_cast<const uint32_t*>(a.v + row * a.ld_v + kv * D)[lane + 32 * i]);
            o[i].x = o[i].x * f + e * v.x;
            o[i].y = o[i].y * f + e * v.y;
        }
    }
    const float inv = any ? 1.f / l : 0.f;
    for (int i = 0; i < N; ++i)
        reinterpret_cast<uint32_t*>(a.out + r * a.ld_out + h * D)[lane + 32 * i] = any ? pack16<DT>(o[i].x * inv, o[i].y * inv) : 0u;
}

const char* attention_error(const mk_paged_cache* cache, int heads) {
    const char* why = cache_error(cache);
    if (!why && cache->head_dim != 64 && cache->head_dim != 128) why = "paged attention: head_dim is 64 or 128";
    if (!why && (heads <= 0 || heads % cache->kv_heads)) why = "paged attention: heads is a multiple of kv_heads";
    return why;
}

}  // namespace
}  // namespace mk

using namespace mk;

extern "C" long long mk_paged_attention_workspace(int device, int heads, const mk_paged_cache* cache, int max_new) {
    const char* why = attention_error(cache, heads);
    return why ? report(MK_E_ARG, why) : 16;
}

extern "C" int mk_paged_attention(int device, const mk_batch* batch, const mk_paged_cache* cache, const void* q, int64_t ld_q, void* out,
                                  int64_t ld_out, int heads, float scale, int window, int max_new, void* workspace, size_t workspace_bytes,
                                  void* stream) {
    const char* why = batch_error(batch);
    if (!why) why = attention_error(cache, heads);
    if (!why && window < 0) why = "paged attention: window is a number of rows (0: the whole context)";
    if (why) return report(MK_E_ARG, why);
    if (batch->rows == 0 || batch->seqs == 0) return MK_OK;
    const long long width = (long long)heads * cache->head_dim;
    if (!q || !out || ld_q < width || ld_out < width || !aligned16(q, ld_q, 2) || !aligned16(out, ld_out, 2))
        return report(MK_E_ARG, "paged attention: rows hold all heads and start on 16-byte boundaries");
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < 16) return report(MK_E_ARG, "paged attention: workspace");
    OnDevice on(device);
    if (!on.ok) return report(MK_E_CUDA, "cudaSetDevice");
    AttnArgs a = {batch_of(batch), pages_of(cache), (const uint16_t*)q, (const uint16_t*)cache->k, (const uint16_t*)cache->v, (uint16_t*)out,
                  ld_q, cache->ld_k, cache->ld_v, ld_out, heads, heads / cache->kv_heads, window, scale * kLog2e};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)batch->rows, (unsigned)((heads + 3) / 4));
    cfg.blockDim = dim3(128);
    cfg.stream = (cudaStream_t)stream;
    cudaError_t e;
    if (cache->dtype == DT_F16)
        e = cache->head_dim == 64 ? cudaLaunchKernelEx(&cfg, attend_row<DT_F16, 64>, a) : cudaLaunchKernelEx(&cfg, attend_row<DT_F16, 128>, a);
    else
        e = cache->head_dim == 64 ? cudaLaunchKernelEx(&cfg, attend_row<DT_BF16, 64>, a) : cudaLaunchKernelEx(&cfg, attend_row<DT_BF16, 128>, a);
    if (e == cudaSuccess) return MK_OK;
    (void)cudaGetLastError();
    return report(MK_E_CUDA, cudaGetErrorString(e));
}

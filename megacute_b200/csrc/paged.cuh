// What the operators over a paged cache share: the packed batch, the page table, 16-bit conversions, and the host side's checks.
#pragma once
#include <cstdio>

#include "mk_device.cuh"

namespace mk {

int report(int code, const char* text);               // (megakernel.cu) remembers `text` for mk_last_cuda_error and returns `code`

// ---- host ----------------------------------------------------------------------------------------------------------------------
// Makes `device` current for the lifetime of the object and puts the caller's device back after.
struct OnDevice {
    int prev = -1;
    bool ok = true;
    explicit OnDevice(int device) {
        if (cudaGetDevice(&prev) != cudaSuccess) { prev = -1; (void)cudaGetLastError(); }
        if (prev == device) prev = -1;                // nothing to put back
        else ok = cudaSetDevice(device) == cudaSuccess;
        if (!ok) { (void)cudaGetLastError(); prev = -1; }
    }
    ~OnDevice() {
        if (prev >= 0) (void)cudaSetDevice(prev);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
};

inline bool aligned16(const void* p, long long ld, int elem_bytes) {
    return ((uintptr_t)p & 15) == 0 && ld >= 0 && (ld * elem_bytes) % 16 == 0;
}
inline int elem_bytes(int dtype) { return dtype == DT_F32 ? 4 : 2; }

// nullptr, or what is wrong
inline const char* batch_error(const mk_batch* b) {
    if (!b || b->rows < 0 || b->seqs < 0) return "batch: rows and seqs are not negative";
    if (b->rows == 0 || b->seqs == 0) return nullptr;
    if (!b->pos || b->pos_ld < 0) return "batch: pos is device memory, one position per sequence";
    if (!b->starts && b->rows % b->seqs) return "batch: without starts every sequence has the same number of rows";
    return nullptr;
}
inline const char* rotation_error(const mk_rotation* r, int head_dim) {
    if (!r || !r->cos || !r->sin || r->rows <= 0) return "rotation: no tables";
    if (r->dtype < DT_BF16 || r->dtype > DT_F16) return "rotation: tables are bf16, fp32 or fp16";
    if (r->columns <= 0 || r->columns % 8 || 2 * r->columns > head_dim) return "rotation: 16, 32, ... elements of a head are rotated, no more than it has";
    const int es = elem_bytes(r->dtype);
    if (!aligned16(r->cos, r->ld_cos, es) || !aligned16(r->sin, r->ld_sin, es)) return "rotation: table rows start on 16-byte boundaries";
    return nullptr;
}
inline const char* cache_error(const mk_paged_cache* c) {
    if (!c || c->pages < 0 || c->table_cols < 0 || (c->pages && (!c->k || !c->v)) || (c->table_cols && !c->table)) return "paged cache: no memory";
    if (c->dtype != DT_BF16 && c->dtype != DT_F16) return "paged cache: bf16 or fp16";
    if (c->page_size < 16 || (c->page_size & (c->page_size - 1))) return "paged cache: page_size is a power of two from 16 up";
    if ((long long)c->pages * c->page_size > 0x7fffffffll) return "paged cache: at most 2^31 - 1 rows";
    if ((long long)c->table_cols * c->page_size > 0x7fff0000ll) return "paged cache: a sequence has at most 2^31 - 65536 rows";
    if (c->table_ld < 0) return "paged cache: table_ld is not negative";
    const long long width = (long long)c->kv_heads * c->head_dim;
    if (c->kv_heads <= 0 || c->head_dim <= 0 || c->ld_k < width || c->ld_v < width) return "paged cache: rows hold kv_heads heads";
    if (!aligned16(c->k, c->ld_k, 2) || !aligned16(c->v, c->ld_v, 2)) return "paged cache: rows start on 16-byte boundaries";
    return nullptr;
}

// ---- device --------------------------------------------------------------------------------------------------------------------
struct Batch {
    const int* pos;
    const int* starts;
    long long pos_ld;
    int rows, seqs, each;                             // each: rows of a sequence where there are no starts
    // first row and number of rows of sequence s, inside the packed batch whatever `starts` holds
    __device__ __forceinline__ int first(int s) const {
        return starts ? min(max(__ldg(starts + s), 0), rows) : s * each;
    }
    __device__ __forceinline__ int count(int s, int r0) const {
        return starts ? min(max(__ldg(starts + s + 1), r0), rows) - r0 : each;
    }
    __device__ __forceinline__ int position(int s) const { return __ldg(pos + s * pos_ld); }
};
inline Batch batch_of(const mk_batch* b) { return Batch{b->pos, b->starts, (long long)b->pos_ld, b->rows, b->seqs, b->rows / b->seqs}; }

// The sequence of row r, -1 if it has none: a whole warp asks for one row, 32 entries of `starts` at a time.
__device__ __forceinline__ int sequence_of_row(const Batch& b, int r) {
    if (!b.starts) return r / b.each;
    const int lane = threadIdx.x & 31;
    int lo = 0, n = b.seqs + 1;                       // entries [lo, lo + n) hold the border; those in front are <= r
    while (n > 0) {
        const int step = (n + 31) / 32, at = lo + lane * step;
        const int below = __popc(__ballot_sync(0xffffffffu, lane * step < n && __ldg(b.starts + at) <= r));
        if (below == 0) break;
        const int skip = (below - 1) * step + 1, left = min(step - 1, n - skip);
        lo += skip;
        n = left;
    }
    return lo > b.seqs ? -1 : lo - 1;                 // (lo: entries <= r)
}

// Kernels are launched with programmatic serialization: their blocks start when those of the kernel in front have ended, and touch no memory before
// this, which waits until its writes can be seen.
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

struct Pages {
    const int* table;
    long long ld;
    int pages, shift, cols;                           // shift: log2 of the page size
    __device__ __forceinline__ int capacity() const { return cols << shift; }
    // first cache row of page `at` of sequence s, -1 if it is absent
    __device__ __forceinline__ int page_row(int s, int at) const {
        if ((unsigned)at >= (unsigned)cols) return -1;
        const int p = __ldg(table + s * ld + at);
        return (unsigned)p < (unsigned)pages ? p << shift : -1;
    }
};
inline Pages pages_of(const mk_paged_cache* c) {
    int shift = 4;
    while ((1 << shift) < c->page_size) ++shift;
    return Pages{c->table, (long long)c->table_ld, c->pages, shift, c->table_cols};
}

template <int DT>
__device__ __forceinline__ float2 unpack16(uint32_t w) {
    if (DT == DT_F16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
    return make_float2(bf16_lo(w), bf16_hi(w));
}
// round to nearest, fp16 beyond its range to infinity
template <int DT>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
    if (DT == DT_F16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

}  // namespace mk

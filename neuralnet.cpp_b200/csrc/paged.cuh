// paged.cuh — what the paged-cache operators share: views of the pool and of the sequences, the place of a position,
// and the checks of arguments.
#pragma once
#include "common.cuh"

namespace nnb {

// bits of dev_flags[1], raised by the kernels and reported by nnb_engine_check
enum { PAGED_BAD_PAGE = 1, PAGED_BAD_LEN = 2, PAGED_NO_ROOM = 4, PAGED_BAD_POS = 8 };

struct PagedView {
    void *k, *v;
    float* w;
    int n_pages, page, heads, dk, pitch;
};
struct SeqView {
    const int32_t *table, *len;
    long long stride;
    int n_seq, max_pages;
};

// index of the row of slot `slot` of a page, -1 if the page is not in the pool
__host__ __device__ inline long long paged_row(int page_id, int n_pages, int heads, int page_size, int head, int slot)
{
    if (page_id < 0 || page_id >= n_pages) return -1;
    return ((long long)page_id * heads + head) * page_size + slot;
}

__host__ __device__ inline int paged_capacity(const PagedView& c, const SeqView& s) { return s.max_pages * c.page; }

#ifdef __CUDACC__
__device__ __forceinline__ void paged_flag(int* flags, int bit) { atomicOr(flags + 1, bit); }

// d_len[s], held inside the table
__device__ __forceinline__ int paged_len(const PagedView& c, const SeqView& s, int seq, int* flags)
{
    const int n = s.len[seq], cap = paged_capacity(c, s);
    if (n >= 0 && n <= cap) return n;
    paged_flag(flags, PAGED_BAD_LEN);
    return n < 0 ? 0 : cap;
}
#endif

nnb_status paged_check_cache(const char* who, const nnb_paged_cache* c, PagedView* out);
nnb_status paged_check_seqs(const char* who, const nnb_paged_cache* c, const nnb_paged_seqs* s, SeqView* out);

// makes the engine's device current for the time of a call
struct DeviceScope {
    int prev = -1;
    bool changed = false;
    explicit DeviceScope(int device)
    {
        if (cudaGetDevice(&prev) == cudaSuccess && prev != device) changed = cudaSetDevice(device) == cudaSuccess;
    }
    ~DeviceScope()
    {
        if (changed) cudaSetDevice(prev);
    }
};

// The operators' kernels are launched with the programmatic attribute: each waits for its predecessor itself, with pdl_wait
// before its first access and in every thread, so that the chain of completions stays whole.
struct PdlOn {
    nnb_engine* e;
    bool prev;
    explicit PdlOn(nnb_engine* en) : e(en), prev(en->pdl) { e->pdl = true; }
    ~PdlOn() { e->pdl = prev; }
};

}  // namespace nnb

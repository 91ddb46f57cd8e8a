// Views of the paged key-value cache shared by its kernels (paged_cache.cu, paged_decode.cu).
#pragma once
#include "tsa_common.cuh"

namespace tsa {

// pools as the kernels see them; element [page][head][slot] of a plane is at ((page * KvHeads + head) << PageShift) + slot
struct TPages {
    uint8_t *K, *V;
    char *KScale, *VScale;
    int *Pos;      // may be null
    float *Weight; // may be null
    int PageCount, PageShift, KvHeads;
    P2D<int> Table;
    int TableCols;
};

// index of a page's plane of one head in units of slots
__device__ __forceinline__ size_t PlaneSlot(const TPages &c, int page, int head)
{
    return (size_t)(unsigned)(page * c.KvHeads + head) << c.PageShift; // page_count * kv_heads fits an int (checked by the host)
}

// tokens a sequence can have: what its table row has room for
__host__ __device__ __forceinline__ long long TableTokens(const TPages &c)
{
    return (long long)c.TableCols << c.PageShift;
}

__device__ __forceinline__ void ClusterArrive()
{
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
}
__device__ __forceinline__ void ClusterWait()
{
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ void ClusterSync()
{
    ClusterArrive();
    ClusterWait();
}
// word of another CTA of the cluster at the place of `mine` in its shared memory
__device__ __forceinline__ unsigned ClusterAddress(const void *mine, int rank)
{
    unsigned r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((unsigned)__cvta_generic_to_shared(mine)), "r"(rank));
    return r;
}

// checks of the arguments that every entry point takes; needVectors: k, v and their scales have to be there
int CheckPages(const char *fn, const tsa_paged_cfg *cfg, const tsa_paged_kv *kv, tsa_ptr2d pageTable, const int *ctxLens, int nSeq, bool needVectors, TPages *res);

} // namespace tsa

// The paged key-value cache: rows in (tsa_paged_append), the choice of an eviction (tsa_paged_evict_select) and the moves that carry it
// out (tsa_paged_evict_move).  The attention over it is in paged_decode.cu.
//
// Layout: a page holds page_size tokens of all key heads, head by head, so that what one head reads of a page is one contiguous block of
// page_size * D bytes of K and as many of V.  All planes (scales, positions, weights) have the same [page][head][slot] order.
#include "paged.cuh"
#include <type_traits>

namespace tsa {

int CheckPages(const char *fn, const tsa_paged_cfg *cfg, const tsa_paged_kv *kv, tsa_ptr2d pageTable, const int *ctxLens, int nSeq, bool needVectors, TPages *res)
{
    TSA_REQUIRE(kv != nullptr, "%s: null cache", fn);
    if (needVectors) {
        TSA_REQUIRE(cfg != nullptr, "%s: null cfg", fn);
        TSA_REQUIRE(cfg->head_dim == 64 || cfg->head_dim == 128, "%s: head_dim %d must be 64 or 128", fn, cfg->head_dim);
        TSA_REQUIRE(cfg->kv_dtype == TSA_I8 || cfg->kv_dtype == TSA_E4M3, "%s: kv dtype must be i8 or e4m3", fn);
        TSA_REQUIRE(cfg->scale_dtype == TSA_F16 || cfg->scale_dtype == TSA_F32, "%s: scale dtype must be f16 or f32", fn);
        TSA_REQUIRE(kv->k && kv->v && kv->k_scale && kv->v_scale, "%s: null k/v/k_scale/v_scale", fn);
        TSA_REQUIRE((uintptr_t)kv->k % 16 == 0 && (uintptr_t)kv->v % 16 == 0 && (uintptr_t)kv->k_scale % 16 == 0 && (uintptr_t)kv->v_scale % 16 == 0,
            "%s: k, v and their scales must be 16-byte aligned", fn);
    }
    TSA_REQUIRE((uintptr_t)kv->pos % 16 == 0 && (uintptr_t)kv->weight % 16 == 0, "%s: pos and weight must be 16-byte aligned", fn);
    int shift = 4;
    while (shift < 8 && (1 << shift) != kv->page_size) {
        ++shift;
    }
    TSA_REQUIRE(kv->page_size == 1 << shift, "%s: page size %d must be 16, 32, 64, 128 or 256", fn, kv->page_size);
    TSA_REQUIRE(kv->page_count > 0 && kv->kv_heads > 0 && (long long)kv->page_count * kv->kv_heads <= 0x7fffffff, "%s: %d pages of %d key heads", fn,
        kv->page_count, kv->kv_heads);
    TSA_REQUIRE(kv->kv_heads <= 65535, "%s: %d key heads (at most 65535)", fn, kv->kv_heads);
    TSA_REQUIRE(nSeq >= 0 && nSeq <= 65535, "%s: %d sequences (at most 65535)", fn, nSeq);
    TSA_REQUIRE(nSeq == 0 || (pageTable.data && ctxLens), "%s: null page table or ctxLens", fn);
    TSA_REQUIRE(nSeq == 0 || (pageTable.ysize >= nSeq && pageTable.xsize > 0), "%s: page table smaller than [nSeq][1]", fn);
    TSA_REQUIRE(nSeq == 0 || (long long)pageTable.xsize << shift <= 1 << 30, "%s: a page table of %d columns has room for more than 2^30 tokens of a sequence", fn,
        pageTable.xsize);
    TSA_REQUIRE((uintptr_t)pageTable.data % 4 == 0 && pageTable.stride_bytes % 4 == 0, "%s: the page table must be 4-byte aligned", fn);
    TPages &c = *res;
    c.K = (uint8_t *)kv->k;
    c.V = (uint8_t *)kv->v;
    c.KScale = (char *)kv->k_scale;
    c.VScale = (char *)kv->v_scale;
    c.Pos = kv->pos;
    c.Weight = kv->weight;
    c.PageCount = kv->page_count;
    c.PageShift = shift;
    c.KvHeads = kv->kv_heads;
    c.Table = P2D<int>(pageTable);
    c.TableCols = pageTable.xsize;
    return TSA_OK;
}

// ---- append ------------------------------------------------------------------------------------------------------------------
struct TAppendParams {
    TPages C;
    const int *CtxLens, *Tokens, *RowStarts;
    int NSeq, Rows;
    int LaneShift; // log2 of the lanes of a row
    P2D<char> KNew, VNew;
    P2D<float> KScaleNew, VScaleNew;
    int *Status;
};

constexpr int APP_AHEAD = 4, APP_MANY_ROWS = 4096;
constexpr int APP_WARPS = 8, APP_MAX_ROWS = 64; // of a CTA: four lanes to a row at least

// The sequence whose rows [starts[s], starts[s + 1]) hold `row`: the last s with starts[s] <= row, -1 if row is in front of all or behind the
// last.  The 2^shift lanes of a row narrow the range by one more than they are per step (sequences without rows have equal starts and are
// stepped over); the warp's rows take as many steps as the one that needs most.
__device__ __forceinline__ int FindSeq(const int *starts, int nSeq, int row, int lane, int shift)
{
    const int lanes = 1 << shift, l = lane & (lanes - 1);
    const unsigned mine = (0xffffffffu >> (32 - lanes)) << (lane - l);
    const bool in = starts[0] <= row && starts[nSeq] > row;
    int lo = 0, hi = in ? nSeq : 1; // starts[lo] <= row < starts[hi]
    while (__any_sync(0xffffffffu, hi - lo > 1)) {
        const int step = (hi - lo + lanes - 1) >> shift;
        const int at = min(lo + (l + 1) * step, hi);
        const bool below = at < hi && starts[at] <= row;
        const int cnt = __popc(__ballot_sync(0xffffffffu, below) & mine);
        hi = min(hi, lo + (cnt + 1) * step);
        lo += cnt * step;
    }
    return in ? lo : -1;
}

// A warp, or a part of one, per row: it finds the row's sequence, slot and page while the row's first 8 pieces of 16 bytes a lane are on their way,
// and stores the heads' pieces.  The warps of a CTA have neighbouring rows, which are neighbours in their page, too: scales, positions and
// weights are stored by all of them, a sector of eight rows at a time (one row at a time, by the row's warp: 42.9 us below instead of 38).
// Bound by the bytes, read once and written once: 9 prompts of 700 .. 4096 rows of 16 heads x 128 with positions and weights, 250 MB, in 38 to 40 us;
// 64 single tokens in 4, which is the host's call.
template <int D, bool SCALE_F16>
__global__ void __launch_bounds__(APP_WARPS * 32) PagedAppendKernel(const TAppendParams p)
{
    constexpr int LPH = D / 16, AHEAD = APP_AHEAD;
    constexpr size_t NOWHERE = ~(size_t)0;
    __shared__ size_t firstOf[APP_MAX_ROWS]; // where the rows' tokens are in the planes of head 0
    __shared__ int posOf[APP_MAX_ROWS];
    const int tid = threadIdx.x, lane = tid & 31;
    const int lanes = 1 << p.LaneShift, l = lane & (lanes - 1), rows = APP_WARPS * 32 >> p.LaneShift; // of the CTA
    const int row0 = blockIdx.x * rows, mine = tid >> p.LaneShift, row = row0 + mine;
    PdlTrigger();
    PdlWait();
    const TPages &c = p.C;
    const int pieces = row < p.Rows ? c.KvHeads * LPH : 0;
    const int4 *ks = nullptr, *vs = nullptr;
    int4 a[AHEAD], b[AHEAD];
    auto load = [&](int i) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            if (i + j * lanes < pieces) {
                a[j] = ks[i + j * lanes]; // not through the read-only path: the kernel before may still write the rows when this one starts
                b[j] = vs[i + j * lanes];
            }
        }
    };
    // the scales that this thread will store: of head h0 and row r of the CTA
    const int r = tid & (rows - 1), h0 = tid / rows;
    float sk = 0, sv = 0;
    if (h0 < c.KvHeads && row0 + r < p.Rows) {
        sk = p.KScaleNew.Row(h0)[row0 + r];
        sv = p.VScaleNew.Row(h0)[row0 + r];
    }
    if (row < p.Rows) {
        ks = reinterpret_cast<const int4 *>(p.KNew.Row(row));
        vs = reinterpret_cast<const int4 *>(p.VNew.Row(row));
    }
    load(l);
    int seq = row < p.Rows ? row : -1, back = 1;
    if (p.RowStarts) {
        seq = FindSeq(p.RowStarts, p.NSeq, row, lane, p.LaneShift);
        back = seq < 0 ? 0 : p.RowStarts[seq + 1] - row;
    }
    size_t first = NOWHERE;
    if (seq >= 0 && row < p.Rows) {
        const int len = p.CtxLens[seq], slot = len - back, col = slot >> c.PageShift;
        int page = -1;
        if (slot >= 0 && col < c.TableCols) {
            page = c.Table.Row(seq)[col];
        }
        if ((unsigned)page < (unsigned)c.PageCount) {
            first = PlaneSlot(c, page, 0) + (slot & ((1 << c.PageShift) - 1)); // the next head's is a page of slots further
            if (l == 0) {
                posOf[mine] = (p.Tokens ? p.Tokens[seq] : len) - back;
            }
        } else if (l == 0 && p.Status) {
            atomicOr(p.Status, kDevBadSpan); // no such place: nothing is stored
        }
    }
    if (l == 0) {
        firstOf[mine] = first;
    }
    if (first != NOWHERE) {
        for (int i = l;;) {
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int x = i + j * lanes;
                if (x < pieces) {
                    const size_t at = (first + ((size_t)(x / LPH) << c.PageShift)) * LPH + x % LPH;
                    reinterpret_cast<int4 *>(c.K)[at] = a[j];
                    reinterpret_cast<int4 *>(c.V)[at] = b[j];
                }
            }
            i += lanes * AHEAD;
            if (i - l >= pieces) {
                break;
            }
            load(i);
        }
    }
    __syncthreads();
    if (firstOf[r] == NOWHERE) {
        return;
    }
    for (int h = h0; h < c.KvHeads; h += APP_WARPS * 32 / rows) {
        const size_t at = firstOf[r] + ((size_t)h << c.PageShift);
        if (h > h0) {
            sk = p.KScaleNew.Row(h)[row0 + r];
            sv = p.VScaleNew.Row(h)[row0 + r];
        }
        if (SCALE_F16) {
            reinterpret_cast<__half *>(c.KScale)[at] = __float2half_rn(sk);
            reinterpret_cast<__half *>(c.VScale)[at] = __float2half_rn(sv);
        } else {
            reinterpret_cast<float *>(c.KScale)[at] = sk;
            reinterpret_cast<float *>(c.VScale)[at] = sv;
        }
        if (c.Pos) {
            c.Pos[at] = posOf[r];
        }
        if (c.Weight) {
            c.Weight[at] = 0.0f;
        }
    }
}

// ---- choice of what stays ----------------------------------------------------------------------------------------------------
struct TSelectParams {
    TPages C;
    const int *CtxLens, *Tokens;
    int NSeq, Keep, Recent, MoveCap;
    int MaxCtx; // the caller's bound of CtxLens
    int Cluster; // CTAs per key head of a sequence
    int2 *Moves; // [nSeq][kvHeads][MoveCap]
    int *Counts; // [nSeq][kvHeads]
    int *NewLens;
    int *Status;
};

constexpr int SEL_BINS = 2048;            // 11, 11 and 10 bits of the order
constexpr int SEL_MAX_CLUSTER = 16, SEL_PORTABLE_CLUSTER = 8;
constexpr int SEL_LIST = 2048;            // orders of a CTA that are counted from a list instead of from all
constexpr int SEL_THREADS = 256;          // of a CTA; or 1024
constexpr int SEL_PER_SM = 4;
constexpr int SEL_AHEAD = 2;              // steps of a warp whose loads are under way together
constexpr int SEL_MAX_SLICE = 44 * 1024;  // slots whose orders fit shared memory

// weights as unsigned integers of the same order; -0 counts as 0, NaN as the greatest; tokens that stay whatever their weight are above all
constexpr unsigned SEL_PINNED = 0xffffffffu, SEL_NAN = 0xfffffffeu;
__device__ __forceinline__ unsigned WeightOrder(float w)
{
    const unsigned b = __float_as_uint(w + 0.0f);
    return w != w ? SEL_NAN : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

// weights and positions of slots slot .. slot + 3 (slot a multiple of 4)
struct TSlotWeights {
    float4 W;
    int4 Pos;
    bool Ok; // the page is in the pool
};
__device__ __forceinline__ int SlotPage(const TSelectParams &p, const int *table, int slot)
{
    return table[slot >> p.C.PageShift];
}
__device__ __forceinline__ TSlotWeights LoadWeights(const TSelectParams &p, int page, int head, int slot)
{
    const TPages &c = p.C;
    TSlotWeights r;
    r.W = make_float4(0, 0, 0, 0);
    r.Pos = make_int4(slot, slot + 1, slot + 2, slot + 3);
    r.Ok = (unsigned)page < (unsigned)c.PageCount;
    if (r.Ok) {
        const size_t at = PlaneSlot(c, page, head) + (slot & ((1 << c.PageShift) - 1));
        r.W = *reinterpret_cast<const float4 *>(c.Weight + at);
        if (p.Recent > 0 && c.Pos) {
            r.Pos = *reinterpret_cast<const int4 *>(c.Pos + at);
        }
    }
    return r;
}
// their orders; slots of pages outside the pool are the lightest
__device__ __forceinline__ uint4 SlotOrders(const TSelectParams &p, const TSlotWeights &x, int newest)
{
    if (!x.Ok) {
        return make_uint4(0, 0, 0, 0);
    }
    uint4 o = make_uint4(WeightOrder(x.W.x), WeightOrder(x.W.y), WeightOrder(x.W.z), WeightOrder(x.W.w));
    if (p.Recent > 0) {
        const int old = newest - p.Recent;
        o.x = x.Pos.x > old ? SEL_PINNED : o.x;
        o.y = x.Pos.y > old ? SEL_PINNED : o.y;
        o.z = x.Pos.z > old ? SEL_PINNED : o.z;
        o.w = x.Pos.w > old ? SEL_PINNED : o.w;
    }
    return o;
}

__device__ __forceinline__ uint4 ClusterLoad16(unsigned address)
{
    uint4 r;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(address) : "memory");
    return r;
}

__device__ __forceinline__ void ClusterAdd(unsigned address, unsigned x)
{
    asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(address), "r"(x) : "memory");
}

template <int WARPS>
struct TSelectShared {
    alignas(16) unsigned Hist[3][SEL_BINS];
    unsigned List[SEL_LIST];  // orders that agree with the first digit
    int ListLen;
    alignas(16) int Found[4]; // bin, how many are still to be taken from it, how many it has
    int4 Total;               // of this CTA: ties, holes, movers
    int4 WarpOf[WARPS];
};

// sum of the values of the warps before this one, and of all (values in shared memory)
template <int WARPS>
__device__ __forceinline__ int WarpsBefore(int mine, int warp, int lane, int *all)
{
    const int v = lane < WARPS ? mine : 0;
    *all = __reduce_add_sync(0xffffffffu, v);
    return __reduce_add_sync(0xffffffffu, lane < warp ? v : 0);
}

// The largest bin at which the sum of the counts from the last bin down reaches `take`: found[0]; how many are to be taken from it: found[1];
// its count: found[2].  One warp: lane l has bins SEL_BINS - 64 (l + 1) .. + 63, then the lane that has the bin looks for it in its own.
__device__ __forceinline__ void FindBin(const unsigned *hist, int lane, int take, int *found)
{
    constexpr int PER = SEL_BINS / 32;
    const int first = SEL_BINS - PER * (lane + 1);
    int mine = 0;
#pragma unroll
    for (int i = 0; i < PER / 4; ++i) {
        const uint4 h = *reinterpret_cast<const uint4 *>(hist + first + 4 * ((i + lane) % (PER / 4))); // turned by the lane: no two in a bank
        mine += (int)(h.x + h.y + h.z + h.w);
    }
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        sum += lane >= o ? v : 0;
    }
    // the lane that has the bin, then its 64 bins two to a lane
    const unsigned reach = __ballot_sync(0xffffffffu, sum >= take);
    const int who = reach ? __ffs(reach) - 1 : 31;
    const int above = __shfl_sync(0xffffffffu, sum - mine, who), base = SEL_BINS - PER * (who + 1);
    const uint2 two = *reinterpret_cast<const uint2 *>(hist + base + PER - 2 * (lane + 1)); // two.y is the larger bin
    const int pair = (int)(two.x + two.y);
    sum = pair;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        sum += lane >= o ? v : 0;
    }
    const int before = above + sum - pair;
    if (before < take && above + sum >= take) {
        const bool larger = before + (int)two.y >= take;
        found[0] = base + PER - 2 * (lane + 1) + (larger ? 1 : 0);
        found[1] = take - before - (larger ? 0 : (int)two.y);
        found[2] = larger ? two.y : two.x;
    }
}

// One cluster of CTAs per (sequence, key head); CTA `rank` has the slots [rank * slice, (rank + 1) * slice), each warp a contiguous run of
// them, four to a lane.  The keep-th largest order is found in three digits: counts of the digit among the orders that agree in the digits
// before (shared memory; a cluster's CTAs add theirs to the first one's, which finds the digit), then the sum from the top.  The orders that agree with
// the first digit are few: they go into a list, which the last digit is counted from.  Ranks in slot order are ballots on top of the
// sums of the warps and CTAs before.  CACHED: the orders stay in shared memory after they are read once.
//
// Not bound by its bytes, 8 per slot read once, but by what depends on one another: page, weight, count, sum, three times over, and the ranks at
// the end.  40 x 8 key heads of 2000 .. 6144 slots: 15 us (2 at the copy's bandwidth); 2 x 4 of 100000 .. 131072: 21 us (1.4).  Of 28 K clocks of the
// former the loads take 6.6 K, each search of a digit 1.1 K, the pass over the second digit 4.8 K, the ranks 2.6 K and the moves 7 K; of the latter each
// digit's exchange 3 to 5 K.  Loads of three, four or six steps ahead instead of two, or three CTAs to an SM instead of four, change nothing.
template <int THREADS, bool CACHED>
__global__ void __launch_bounds__(THREADS, THREADS == SEL_THREADS ? SEL_PER_SM : 1) PagedSelectKernel(const TSelectParams p)
{
    constexpr int WARPS = THREADS / 32;
    extern __shared__ uint4 cached[];
    __shared__ __align__(16) TSelectShared<WARPS> sh;
    const int head = blockIdx.x / p.Cluster, rank = blockIdx.x % p.Cluster, seq = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned below = (1u << lane) - 1;
    const TPages &c = p.C;
    PdlTrigger();
    for (int i = tid; i < 3 * SEL_BINS / 4; i += THREADS) {
        reinterpret_cast<uint4 *>(sh.Hist)[i] = make_uint4(0, 0, 0, 0);
    }
    if (tid == 0) {
        sh.ListLen = 0;
    }
    PdlWait();
    const int len = p.CtxLens[seq];
    const size_t unit = (size_t)seq * c.KvHeads + head;
    int2 *moves = p.Moves + unit * p.MoveCap;
    const bool tooLong = len > p.MaxCtx || len > TableTokens(c);
    const bool none = len <= p.Keep || tooLong;
    if (tid == 0 && rank == 0) {
        if (tooLong && p.Status) {
            atomicOr(p.Status, kDevBadSpan);
        }
        if (head == 0) {
            p.NewLens[seq] = none ? len : p.Keep;
        }
        if (none) {
            p.Counts[unit] = 0;
        }
    }
    if (none) { // the same in all CTAs of the cluster
        for (int i = rank * THREADS + tid; i < p.MoveCap; i += p.Cluster * THREADS) {
            moves[i] = make_int2(-1, -1);
        }
        return;
    }
    const int *table = c.Table.Row(seq);
    const int newest = (p.Tokens ? p.Tokens[seq] : len) - 1;
    // slots of a CTA and of a warp: equal parts of what the sequence has, in whole steps of 128
    const int warps = p.Cluster * WARPS;
    const int per = ((len + warps - 1) / warps + 127) & ~127;
    const int slice = per * WARPS;
    const int beg = min(rank * slice + warp * per, len), end = min(beg + per, len);
    bool bad = false;
    auto orders = [&](int s) {
        if (CACHED) {
            return cached[(s - rank * slice) >> 2];
        }
        return SlotOrders(p, LoadWeights(p, SlotPage(p, table, s), head, s), newest);
    };
    // one more in the bin of each order that is in: (order >> shift) & low; equal bins of a whole step (weights that are all zero) are one addition
    auto count = [&](unsigned *hist, const uint4 &o, int shift, unsigned low, unsigned in) {
        const unsigned x = o.x >> shift & low, y = o.y >> shift & low, z = o.z >> shift & low, w = o.w >> shift & low;
        if (__all_sync(0xffffffffu, in == 15 && x == y && x == z && x == w)) {
            const unsigned first = __shfl_sync(0xffffffffu, x, 0);
            if (__all_sync(0xffffffffu, x == first)) {
                if (lane == 0) {
                    atomicAdd(hist + first, 128);
                }
                return;
            }
        }
        if (in & 1) {
            atomicAdd(hist + x, 1);
        }
        if (in & 2) {
            atomicAdd(hist + y, 1);
        }
        if (in & 4) {
            atomicAdd(hist + z, 1);
        }
        if (in & 8) {
            atomicAdd(hist + w, 1);
        }
    };
    // of four slots from s on, the ones below `limit`
    auto until = [](int s, int limit) { return (1u << max(0, min(4, limit - s))) - 1; };
    // of four orders, the ones that agree with the digits found so far
    auto agree = [](const uint4 &o, unsigned mask, unsigned cut) {
        return (unsigned)((o.x & mask) == cut) | (unsigned)((o.y & mask) == cut) << 1 | (unsigned)((o.z & mask) == cut) << 2 | (unsigned)((o.w & mask) == cut) << 3;
    };
    __syncthreads(); // the counts are zero
    if (p.Cluster > 1) {
        ClusterArrive();
    }
    for (int s0 = beg; s0 < end; s0 += 128 * SEL_AHEAD) {
        int page[SEL_AHEAD];
        TSlotWeights x[SEL_AHEAD];
#pragma unroll
        for (int j = 0; j < SEL_AHEAD; ++j) {
            const int s = s0 + 128 * j + 4 * lane;
            page[j] = s < end ? SlotPage(p, table, s) : -1;
        }
#pragma unroll
        for (int j = 0; j < SEL_AHEAD; ++j) {
            x[j] = LoadWeights(p, page[j], head, s0 + 128 * j + 4 * lane);
        }
#pragma unroll
        for (int j = 0; j < SEL_AHEAD; ++j) {
            const int s = s0 + 128 * j + 4 * lane;
            if (s0 + 128 * j >= end) {
                break;
            }
            const uint4 o = SlotOrders(p, x[j], newest);
            if (s < end) {
                bad |= !x[j].Ok;
                if (CACHED) {
                    cached[(s - rank * slice) >> 2] = o;
                }
            }
            count(sh.Hist[0], o, 21, 2047, until(s, end));
        }
    }
    unsigned cut = 0;     // the digits found so far
    int take = p.Keep;    // how many of the orders that agree with them stay
    int equal = 0;        // how many agree
#pragma unroll
    for (int digit = 0; digit < 3; ++digit) {
        constexpr int SHIFT[3] = {21, 10, 0};
        constexpr unsigned low = 1023;
        if (digit == 1) {
#pragma unroll 2
            for (int s0 = beg; s0 < end; s0 += 128) {
                const int s = s0 + 4 * lane;
                const uint4 o4 = s < end ? orders(s) : make_uint4(0, 0, 0, 0);
                const unsigned in = until(s, end) & agree(o4, 0xffe00000u, cut);
                if (in) {
                    const unsigned o[4] = {o4.x, o4.y, o4.z, o4.w};
                    int at = atomicAdd(&sh.ListLen, __popc(in));
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (in >> i & 1) {
                            if (at < SEL_LIST) {
                                sh.List[at] = o[i];
                            }
                            ++at;
                        }
                    }
                }
                count(sh.Hist[1], o4, 10, 2047, in);
            }
        } else if (digit == 2) {
            if (sh.ListLen <= SEL_LIST) {
                for (int i = tid; i < sh.ListLen; i += THREADS) {
                    const unsigned o = sh.List[i];
                    if ((o & 0xfffffc00u) == cut) {
                        atomicAdd(&sh.Hist[2][o & 1023], 1);
                    }
                }
            } else {
                for (int s0 = beg; s0 < end; s0 += 128) {
                    const int s = s0 + 4 * lane;
                    const uint4 o = s < end ? orders(s) : make_uint4(0, 0, 0, 0);
                    count(sh.Hist[2], o, 0, low, until(s, end) & agree(o, 0xfffffc00u, cut));
                }
            }
        }
        __syncthreads();
        if (p.Cluster > 1) {
            // the first CTA's counts become those of the cluster
            if (digit == 0) {
                ClusterWait(); // they were zero
            }
            if (rank > 0) {
                for (int i = tid; i < SEL_BINS; i += THREADS) {
                    const unsigned n = sh.Hist[digit][i];
                    if (n) {
                        ClusterAdd(ClusterAddress(&sh.Hist[digit][i], 0), n);
                    }
                }
            }
            ClusterSync();
        }
        if (rank == 0 && warp == 0) {
            FindBin(sh.Hist[digit], lane, take, sh.Found);
        }
        if (p.Cluster > 1) {
            ClusterSync();
            const uint4 found = ClusterLoad16(ClusterAddress(sh.Found, 0));
            cut |= found.x << SHIFT[digit];
            take = (int)found.y;
            equal = (int)found.z;
        } else {
            __syncthreads();
            cut |= (unsigned)sh.Found[0] << SHIFT[digit];
            take = sh.Found[1];
            equal = sh.Found[2];
        }
    }
    // `take` of the orders equal to cut stay, the first ones in slot order; mostly that is all of them
    const bool allTies = equal == take;
    int ties = take;
    if (!allTies) {
        int n = 0;
        for (int s0 = beg; s0 < end; s0 += 128) {
            const int s = s0 + 4 * lane;
            if (s < end) {
                const uint4 o = orders(s);
                n += (o.x == cut) + (s + 1 < end && o.y == cut) + (s + 2 < end && o.z == cut) + (s + 3 < end && o.w == cut);
            }
        }
        n = __reduce_add_sync(0xffffffffu, n);
        if (lane == 0) {
            sh.WarpOf[warp].x = n;
        }
        __syncthreads();
        int total;
        int before = WarpsBefore<WARPS>(lane < WARPS ? sh.WarpOf[lane].x : 0, warp, lane, &total);
        if (p.Cluster > 1) {
            if (tid == 0) {
                sh.Total.x = total;
            }
            ClusterSync();
            for (int r = 0; r < rank; ++r) {
                before += (int)ClusterLoad16(ClusterAddress(&sh.Total, r)).x;
            }
        }
        ties -= before; // left for this warp's slots
    }
    // one slot per lane from here on
    auto order = [&](int s) {
        if (CACHED) {
            return reinterpret_cast<const unsigned *>(cached)[s - rank * slice];
        }
        const uint4 o = orders(s & ~3);
        return s & 2 ? (s & 1 ? o.w : o.z) : (s & 1 ? o.y : o.x);
    };
    // whether slot s, of order o, stays; `left`: of the ties
    auto kept = [&](int s, unsigned o, int &left) {
        bool k = s < end && o >= cut;
        if (!allTies) {
            const unsigned tie = __ballot_sync(0xffffffffu, k && o == cut);
            k = k && (o > cut || __popc(tie & below) < left);
            left -= __popc(tie);
        }
        return k;
    };
    // slots that leave a hole in front of the budget, or that are moved from behind it
    int hole = 0, mover = 0, left = ties;
    for (int s0 = beg; s0 < end; s0 += 128) {
        unsigned o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int s = s0 + 32 * j + lane;
            o[j] = s < end ? order(s) : 0;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int s = s0 + 32 * j + lane;
            const bool k = kept(s, o[j], left);
            hole += s < p.Keep && s < end && !k;
            mover += s >= p.Keep && k;
        }
    }
    hole = __reduce_add_sync(0xffffffffu, hole);
    mover = __reduce_add_sync(0xffffffffu, mover);
    __syncthreads(); // WarpOf has been read
    if (lane == 0) {
        sh.WarpOf[warp] = make_int4(0, hole, mover, 0);
    }
    __syncthreads();
    const int4 of = lane < WARPS ? sh.WarpOf[lane] : make_int4(0, 0, 0, 0);
    int4 total = make_int4(0, 0, 0, 0);
    hole = WarpsBefore<WARPS>(of.y, warp, lane, &total.y);
    mover = WarpsBefore<WARPS>(of.z, warp, lane, &total.z);
    int moved = total.z;
    if (p.Cluster > 1) {
        ClusterSync(); // the ties of Total have been read
        if (tid == 0) {
            sh.Total = total;
        }
        ClusterSync();
        uint4 x = make_uint4(0, 0, 0, 0);
        if (lane < p.Cluster) {
            x = ClusterLoad16(ClusterAddress(&sh.Total, lane));
        }
        moved = __reduce_add_sync(0xffffffffu, (int)x.z);
        hole += __reduce_add_sync(0xffffffffu, lane < rank ? (int)x.y : 0);
        mover += __reduce_add_sync(0xffffffffu, lane < rank ? (int)x.z : 0);
    }
    // (as many of each as there is room for: at most min(keep, len - keep))
    left = ties;
    for (int s0 = beg; s0 < end; s0 += 128) {
        unsigned o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int s = s0 + 32 * j + lane;
            o[j] = s < end ? order(s) : 0;
        }
        if (s0 < p.Keep && s0 + 128 > p.Keep) {
            // the budget ends in this step
#pragma unroll 1
            for (int j = 0; j < 4; ++j) {
                const int s = s0 + 32 * j + lane;
                const bool k = kept(s, s < end ? order(s) : 0, left), isHole = s < p.Keep && s < end && !k, isMover = s >= p.Keep && k;
                const unsigned holes = __ballot_sync(0xffffffffu, isHole), movers = __ballot_sync(0xffffffffu, isMover);
                if (isHole) {
                    moves[hole + __popc(holes & below)].x = s;
                }
                if (isMover) {
                    moves[mover + __popc(movers & below)].y = s;
                }
                hole += __popc(holes);
                mover += __popc(movers);
            }
            continue;
        }
        // all in front of it or all behind it
        const bool front = s0 < p.Keep;
        int *const dst = front ? &moves[0].x : &moves[0].y;
        int &sofar = front ? hole : mover;
        unsigned which[4];
        bool is[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int s = s0 + 32 * j + lane;
            const bool k = kept(s, o[j], left);
            is[j] = front ? s < end && !k : k;
            which[j] = __ballot_sync(0xffffffffu, is[j]);
        }
        int at = sofar;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (is[j]) {
                dst[2 * (at + __popc(which[j] & below))] = s0 + 32 * j + lane;
            }
            at += __popc(which[j]);
        }
        sofar = at;
    }
    for (int i = moved + rank * THREADS + tid; i < p.MoveCap; i += p.Cluster * THREADS) {
        moves[i] = make_int2(-1, -1);
    }
    if (tid == 0 && rank == 0) {
        p.Counts[unit] = moved;
    }
    if (bad && p.Status) {
        atomicOr(p.Status, kDevBadSpan);
    }
    if (p.Cluster > 1) {
        ClusterSync(); // no CTA leaves while another reads its shared memory
    }
}

// CTAs of a key head, their threads and slots: the least of what the forms are expected to take, in ns.  Measured on 8 .. 1024 key heads of
// 256 .. 64000 slots: a CTA alone on its SM takes 4.6 us and 1.28 ns a slot with 256 threads, 5.8 us and 0.65 ns with 1024 (1.6 ns where it
// reads the weights again in every pass); the exchange inside a cluster 4.5 us, of sixteen CTAs 10; CTAs that share an SM slow each other by 30 to
// 50 %.  What comes of it, in us: 8 heads of 1000 slots 5.8 with 256 threads, 6.7 with 1024; of 4000 10.0 and 7.9; of 64000 in 8 CTAs 20.9 and 16.6,
// in one 100; of 400000 in 8 CTAs 94, in 16 63, of 6 heads 34; 256 heads of 4000 13.5 and 15.4.
struct TSelectForm {
    int Threads, Cluster, Slice;
};
static TSelectForm SelectForm(long long units, int longest, int sms)
{
    TSelectForm best = {};
    long long least = 0;
    for (int threads = SEL_THREADS; threads <= 1024; threads += 1024 - SEL_THREADS) {
        for (int cluster = 1; cluster <= SEL_MAX_CLUSTER; cluster *= 2) {
            const bool many = threads > SEL_THREADS;
            const int warps = cluster * threads / 32, slice = ((longest + warps - 1) / warps + 127) / 128 * 128 * (threads / 32);
            const bool cached = slice <= SEL_MAX_SLICE;
            const int room = 227 * 1024 / (int)((many ? sizeof(TSelectShared<32>) : sizeof(TSelectShared<SEL_THREADS / 32>)) + 1024 + (cached ? 4 * slice : 0));
            const int perSm = many ? 1 : room < SEL_PER_SM ? room : SEL_PER_SM;
            const bool sixteen = cluster > SEL_PORTABLE_CLUSTER;
            if (!many && (!cached || sixteen)) {
                continue; // 1024 threads read twice as fast
            }
            // SMs that clusters find place on: all of a cluster have to be in one part of the chip.  Of CTAs that have an SM each, 74 clusters of two ran at
            // once, 33 of four (35 in two waves), 15 of eight and 6 of sixteen
            const int used = cluster <= 2 ? sms : cluster == 4 ? 132 : cluster == 8 ? (many ? 120 : 128) : 96;
            const long long ctas = units * cluster, onSm = (ctas + used - 1) / used, waves = (onSm + perSm - 1) / perSm;
            const long long alone = (many ? 5800 + (cached ? 65ll : 160ll) * slice / 100 : 4600 + 128ll * slice / 100) + (sixteen ? 10000 : cluster > 1 ? 4500 : 0);
            const long long sharing = onSm < perSm ? onSm : perSm;
            const long long time = waves * alone * (sharing == 1 ? 10 : 12 + sharing / 2) / 10;
            if (least == 0 || time < least) {
                least = time;
                best = {threads, cluster, slice};
            }
        }
    }
    return best;
}

// ---- the moves ---------------------------------------------------------------------------------------------------------------
struct TMoveParams {
    TPages C;
    const int2 *Moves;
    const int *Counts;
    int NSeq, MoveCap;
    int *Status;
};

constexpr int MOV_WARPS = 4;

// A warp takes 32 moves: each lane looks up the pages of one and carries its scales, position and weight; then 2 D / 16 lanes at a time
// carry a row of K and V, MOV_AHEAD rows of a lane on their way together (46.9 us below with one).  Sources and destinations of a head are
// different slots (sources lie behind the budget), so no order is needed.  Bound by rows of 64 or 128 bytes and by planes of which a sector of 32 bytes is
// moved for 2 or 4: 40 caches of 8 heads x 128 cut from up to 6144 to 2048 slots, 180 MB without that, in 39 us.
constexpr int MOV_AHEAD = 8;
template <int D, int SCALE_BYTES>
__global__ void __launch_bounds__(MOV_WARPS * 32) PagedMoveKernel(const TMoveParams p)
{
    typedef typename std::conditional<SCALE_BYTES == 2, uint16_t, uint32_t>::type TScale;
    constexpr int LPM = 2 * D / 16, PER = 32 / LPM; // lanes per move, moves per step
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int head = blockIdx.y, seq = blockIdx.z;
    PdlTrigger();
    PdlWait();
    const TPages &c = p.C;
    const size_t unit = (size_t)seq * c.KvHeads + head;
    const int base = (blockIdx.x * MOV_WARPS + warp) * 32;
    const int2 *moves = p.Moves + unit * p.MoveCap;
    const int count = min(p.Counts[unit], p.MoveCap);
    if (base >= count) {
        return;
    }
    const int *table = c.Table.Row(seq);
    const int mask = (1 << c.PageShift) - 1;
    bool ok = base + lane < count;
    size_t to = 0, of = 0;
    if (ok) {
        const int2 m = moves[base + lane];
        const long long room = TableTokens(c);
        ok = m.x >= 0 && m.y >= 0 && m.x < room && m.y < room;
        if (ok) {
            const int pt = table[m.x >> c.PageShift], pf = table[m.y >> c.PageShift];
            ok = (unsigned)pt < (unsigned)c.PageCount && (unsigned)pf < (unsigned)c.PageCount;
            if (ok) {
                to = PlaneSlot(c, pt, head) + (m.x & mask);
                of = PlaneSlot(c, pf, head) + (m.y & mask);
            }
        }
        if (!ok && p.Status) {
            atomicOr(p.Status, kDevBadSpan);
        }
    }
    const unsigned okMask = __ballot_sync(0xffffffffu, ok);
    TScale sk = 0, sv = 0;
    int pos = 0;
    float weight = 0;
    if (ok) {
        sk = reinterpret_cast<const TScale *>(c.KScale)[of];
        sv = reinterpret_cast<const TScale *>(c.VScale)[of];
        pos = c.Pos ? c.Pos[of] : 0;
        weight = c.Weight ? c.Weight[of] : 0.0f;
    }
    const int sub = lane % LPM;
    int4 *const pool = reinterpret_cast<int4 *>(sub < D / 16 ? c.K : c.V);
    const int piece = sub % (D / 16);
#pragma unroll 1
    for (int i = 0; i < 32 && okMask >> i; i += PER * MOV_AHEAD) {
        int4 x[MOV_AHEAD];
#pragma unroll
        for (int j = 0; j < MOV_AHEAD; ++j) {
            const int m = i + j * PER + lane / LPM;
            const size_t f = __shfl_sync(0xffffffffu, of, m & 31);
            if (okMask >> (m & 31) & 1) {
                x[j] = pool[f * (D / 16) + piece];
            }
        }
#pragma unroll
        for (int j = 0; j < MOV_AHEAD; ++j) {
            const int m = i + j * PER + lane / LPM;
            const size_t t = __shfl_sync(0xffffffffu, to, m & 31);
            if (okMask >> (m & 31) & 1) {
                pool[t * (D / 16) + piece] = x[j];
            }
        }
    }
    if (ok) {
        reinterpret_cast<TScale *>(c.KScale)[to] = sk;
        reinterpret_cast<TScale *>(c.VScale)[to] = sv;
        if (c.Pos) {
            c.Pos[to] = pos;
        }
        if (c.Weight) {
            c.Weight[to] = weight;
        }
    }
}

static bool Overlap(const void *a, size_t aBytes, const void *b, size_t bBytes)
{
    return a && b && (uintptr_t)a < (uintptr_t)b + bBytes && (uintptr_t)b < (uintptr_t)a + aBytes;
}

} // namespace tsa

using namespace tsa;

extern "C" __attribute__((visibility("default"))) int tsa_paged_append(const tsa_paged_cfg *cfg, const tsa_paged_kv *kv, tsa_ptr2d pageTable,
    const int *ctxLens, const int *tokens, const int *rowStarts, int nSeq, int rows, tsa_ptr2d kNew, tsa_ptr2d kScaleNew, tsa_ptr2d vNew, tsa_ptr2d vScaleNew,
    int *statusWord, tsa_stream_t stream)
{
    TAppendParams p;
    int rc = CheckPages("tsa_paged_append", cfg, kv, pageTable, ctxLens, nSeq, true, &p.C);
    if (rc != TSA_OK) {
        return rc;
    }
    TSA_REQUIRE(rows >= 0, "tsa_paged_append: negative row count");
    TSA_REQUIRE(rowStarts || rows <= nSeq, "tsa_paged_append: %d rows of %d sequences without rowStarts", rows, nSeq);
    if (rows == 0 || nSeq == 0) {
        return TSA_OK;
    }
    const int rowBytes = kv->kv_heads * cfg->head_dim;
    TSA_REQUIRE((long long)kv->kv_heads * cfg->head_dim <= 0x7fffffff, "tsa_paged_append: %d key heads", kv->kv_heads);
    TSA_REQUIRE(kNew.data && vNew.data && kScaleNew.data && vScaleNew.data, "tsa_paged_append: null kNew/vNew/kScaleNew/vScaleNew");
    TSA_REQUIRE(kNew.xsize >= rowBytes && vNew.xsize >= rowBytes && kNew.ysize >= rows && vNew.ysize >= rows, "tsa_paged_append: kNew/vNew extents");
    TSA_REQUIRE((uintptr_t)kNew.data % 16 == 0 && kNew.stride_bytes % 16 == 0 && (uintptr_t)vNew.data % 16 == 0 && vNew.stride_bytes % 16 == 0,
        "tsa_paged_append: kNew/vNew must be 16-byte aligned");
    TSA_REQUIRE(kScaleNew.xsize >= rows && vScaleNew.xsize >= rows && kScaleNew.ysize >= kv->kv_heads && vScaleNew.ysize >= kv->kv_heads,
        "tsa_paged_append: kScaleNew/vScaleNew must be [kvHeads][rows]");
    TSA_REQUIRE((uintptr_t)kScaleNew.data % 4 == 0 && kScaleNew.stride_bytes % 4 == 0 && (uintptr_t)vScaleNew.data % 4 == 0 && vScaleNew.stride_bytes % 4 == 0,
        "tsa_paged_append: scale planes must be 4-byte aligned");
    p.CtxLens = ctxLens;
    p.Tokens = tokens;
    p.RowStarts = rowStarts;
    p.NSeq = nSeq;
    p.Rows = rows;
    p.KNew = P2D<char>(kNew);
    p.VNew = P2D<char>(vNew);
    p.KScaleNew = P2D<float>(kScaleNew);
    p.VScaleNew = P2D<float>(vScaleNew);
    p.Status = statusWord;
    // Lanes of a row: a piece for each, or, where there are rows enough to fill the device, as many as they can have under way.  Measured, in us, by
    // pieces a lane (1, 4; a whole warp for each row): 200000 rows of one head x 128 26.8, 19.4 (81), of 4 x 64 51.7, 35.6 (84), of 12 x 64 118, 101 (118);
    // 64 rows of 4 x 64 2.5, 3.6 (2.4), 1024 of them 3.3, 4.1 (3.1)
    const int most = rows < APP_MANY_ROWS ? 1 : APP_AHEAD;
    p.LaneShift = 2;
    while (p.LaneShift < 5 && (most << p.LaneShift) < rowBytes / 16) {
        ++p.LaneShift;
    }
    const bool f16 = cfg->scale_dtype == TSA_F16;
    const void *kern = cfg->head_dim == 128 ? (f16 ? (const void *)PagedAppendKernel<128, true> : (const void *)PagedAppendKernel<128, false>)
                                            : (f16 ? (const void *)PagedAppendKernel<64, true> : (const void *)PagedAppendKernel<64, false>);
    void *args[] = {&p};
    return CheckCuda(LaunchPdl(kern, dim3((rows - 1) / (APP_WARPS * 32 >> p.LaneShift) + 1), dim3(APP_WARPS * 32), 0, (cudaStream_t)stream, args), "tsa_paged_append launch");
}

extern "C" __attribute__((visibility("default"))) int tsa_paged_evict_select(const tsa_paged_kv *kv, tsa_ptr2d pageTable, const int *ctxLens, const int *tokens,
    int nSeq, int maxCtx, int keep, int recent, int *moves, int moveCap, int *moveCounts, int *newLens, int *statusWord, tsa_stream_t stream)
{
    TSelectParams p;
    int rc = CheckPages("tsa_paged_evict_select", nullptr, kv, pageTable, ctxLens, nSeq, false, &p.C);
    if (rc != TSA_OK) {
        return rc;
    }
    TSA_REQUIRE(kv->weight != nullptr, "tsa_paged_evict_select: the cache keeps no weights");
    TSA_REQUIRE(maxCtx >= 0 && keep >= 1 && recent >= 0 && recent <= keep, "tsa_paged_evict_select: keep %d of at most %d tokens, %d of them the newest", keep,
        maxCtx, recent);
    TSA_REQUIRE((kv->pos == nullptr) == (tokens == nullptr), "tsa_paged_evict_select: positions and the sequences' token counts go together");
    if (nSeq == 0) {
        return TSA_OK;
    }
    const int most = maxCtx - keep < keep ? maxCtx - keep : keep;
    TSA_REQUIRE(moves && moveCounts && newLens, "tsa_paged_evict_select: null moves/moveCounts/newLens");
    TSA_REQUIRE(moveCap >= 1 && moveCap >= most, "tsa_paged_evict_select: room for %d moves of a head needed, %d given", most < 1 ? 1 : most, moveCap);
    TSA_REQUIRE((uintptr_t)moves % 8 == 0, "tsa_paged_evict_select: moves must be 8-byte aligned");
    // a CTA of one key head may write its part before another has read the lengths
    const size_t counts = (size_t)nSeq * kv->kv_heads * sizeof(int), lens = (size_t)nSeq * sizeof(int);
    for (const int *in : {ctxLens, tokens}) {
        TSA_REQUIRE(!Overlap(newLens, lens, in, lens) && !Overlap(moveCounts, counts, in, lens) && !Overlap(moves, counts * moveCap * 2, in, lens),
            "tsa_paged_evict_select: moves, moveCounts and newLens must not overlap ctxLens or tokens");
    }
    p.CtxLens = ctxLens;
    p.Tokens = tokens;
    p.NSeq = nSeq;
    p.Keep = keep;
    p.Recent = recent;
    p.MoveCap = moveCap;
    p.MaxCtx = maxCtx;
    p.Moves = (int2 *)moves;
    p.Counts = moveCounts;
    p.NewLens = newLens;
    p.Status = statusWord;
    const long long room = TableTokens(p.C);
    const int longest = room < maxCtx ? (int)room : maxCtx;
    int dev = 0, sms = 0;
    rc = CheckCuda(cudaGetDevice(&dev), "cudaGetDevice");
    if (rc == TSA_OK) {
        rc = CheckCuda(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev), "cudaDeviceGetAttribute");
    }
    if (rc != TSA_OK) {
        return rc;
    }
    const TSelectForm form = SelectForm((long long)kv->kv_heads * nSeq, longest, sms);
    p.Cluster = form.Cluster;
    const int threads = form.Threads, slice = form.Slice;
    const bool many = threads > SEL_THREADS, cached = slice <= SEL_MAX_SLICE;
    const void *kern = many ? (cached ? (const void *)PagedSelectKernel<1024, true> : (const void *)PagedSelectKernel<1024, false>)
                            : (const void *)PagedSelectKernel<SEL_THREADS, true>;
    const size_t smem = cached ? (size_t)slice * sizeof(unsigned) : 0;
    if (smem > 8 * 1024) { // beyond 48 KB with the counts.  The same limit in every call: another thread's may come between this and the launch
        rc = CheckCuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SEL_MAX_SLICE * sizeof(unsigned)), "cudaFuncSetAttribute");
        if (rc != TSA_OK) {
            return rc;
        }
    }
    if (p.Cluster > SEL_PORTABLE_CLUSTER) {
        rc = CheckCuda(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "cudaFuncSetAttribute");
        if (rc != TSA_OK) {
            return rc;
        }
    }
    void *args[] = {&p};
    return CheckCuda(LaunchPdl(kern, dim3(kv->kv_heads * p.Cluster, nSeq), dim3(threads), smem, (cudaStream_t)stream, args, p.Cluster),
        "tsa_paged_evict_select launch");
}

extern "C" __attribute__((visibility("default"))) int tsa_paged_evict_move(const tsa_paged_cfg *cfg, const tsa_paged_kv *kv, tsa_ptr2d pageTable,
    const int *moves, int moveCap, const int *moveCounts, int nSeq, int *statusWord, tsa_stream_t stream)
{
    TMoveParams p;
    int rc = CheckPages("tsa_paged_evict_move", cfg, kv, pageTable, moveCounts, nSeq, true, &p.C);
    if (rc != TSA_OK) {
        return rc;
    }
    TSA_REQUIRE(moveCap >= 0, "tsa_paged_evict_move: negative moveCap");
    if (nSeq == 0 || moveCap == 0) {
        return TSA_OK;
    }
    TSA_REQUIRE(moves != nullptr && (uintptr_t)moves % 8 == 0, "tsa_paged_evict_move: moves missing or not 8-byte aligned");
    p.Moves = (const int2 *)moves;
    p.Counts = moveCounts;
    p.NSeq = nSeq;
    p.MoveCap = moveCap;
    p.Status = statusWord;
    const bool f16 = cfg->scale_dtype == TSA_F16;
    const void *kern = cfg->head_dim == 128 ? (f16 ? (const void *)PagedMoveKernel<128, 2> : (const void *)PagedMoveKernel<128, 4>)
                                            : (f16 ? (const void *)PagedMoveKernel<64, 2> : (const void *)PagedMoveKernel<64, 4>);
    void *args[] = {&p};
    const int per = MOV_WARPS * 32;
    return CheckCuda(LaunchPdl(kern, dim3((moveCap + per - 1) / per, kv->kv_heads, nSeq), dim3(MOV_WARPS * 32), 0, (cudaStream_t)stream, args),
        "tsa_paged_evict_move launch");
}

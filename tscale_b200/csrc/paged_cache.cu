// The paged key-value cache: rows in (tsa_paged_append), the choice of an eviction (tsa_paged_evict_select) and the moves that carry it
// out (tsa_paged_evict_move).  The attention over it is in paged_decode.cu.
//
// Layout: a page holds page_size tokens of all key heads, head by head, so that what one head reads of a page is one contiguous block of
// page_size * D bytes of K and as many of V.  All planes (scales, positions, weights) have the same [page][head][slot] order.
#include "paged.cuh"

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
    TSA_REQUIRE(nSeq >= 0 && nSeq <= 65535, "%s: %d sequences (at most 65535)", fn, nSeq);
    TSA_REQUIRE(nSeq == 0 || (pageTable.data && ctxLens), "%s: null page table or ctxLens", fn);
    TSA_REQUIRE(nSeq == 0 || (pageTable.ysize >= nSeq && pageTable.xsize > 0), "%s: page table smaller than [nSeq][1]", fn);
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
    P2D<char> KNew, VNew;
    P2D<float> KScaleNew, VScaleNew;
    int *Status;
};

constexpr int APP_WARPS = 4;

// the sequence whose rows [starts[s], starts[s + 1]) hold `row`: the last s with starts[s] <= row, -1 if row is in front of all or behind the
// last.  A warp narrows the range by 33 per step (sequences without rows have equal starts and are stepped over).
__device__ __forceinline__ int FindSeq(const int *starts, int nSeq, int row, int lane)
{
    if (starts[0] > row || starts[nSeq] <= row) {
        return -1;
    }
    int lo = 0, hi = nSeq; // starts[lo] <= row < starts[hi]
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int at = min(lo + (lane + 1) * step, hi);
        const bool below = at < hi && starts[at] <= row;
        const int cnt = __popc(__ballot_sync(0xffffffffu, below));
        hi = min(hi, lo + (cnt + 1) * step);
        lo += cnt * step;
    }
    return lo;
}

// One warp per row: it finds the row's sequence, slot and page, and copies the row's heads 16 bytes a lane.
template <int D, bool SCALE_F16>
__global__ void __launch_bounds__(APP_WARPS * 32) PagedAppendKernel(const TAppendParams p)
{
    constexpr int LPH = D / 16;
    const int lane = threadIdx.x & 31;
    const int row = blockIdx.x * APP_WARPS + (threadIdx.x >> 5);
    PdlTrigger();
    PdlWait();
    if (row >= p.Rows) {
        return;
    }
    int seq = row, back = 1;
    if (p.RowStarts) {
        seq = FindSeq(p.RowStarts, p.NSeq, row, lane);
        if (seq < 0) {
            return;
        }
        back = p.RowStarts[seq + 1] - row;
    }
    const TPages &c = p.C;
    const int slot = p.CtxLens[seq] - back;
    const int col = slot >> c.PageShift;
    int page = -1;
    if (slot >= 0 && col < c.TableCols) {
        page = c.Table.Row(seq)[col];
    }
    if (page < 0 || page >= c.PageCount) {
        if (lane == 0 && p.Status) {
            atomicOr(p.Status, kDevBadSpan); // no such place: nothing is stored
        }
        return;
    }
    const int inPage = slot & ((1 << c.PageShift) - 1);
    const size_t first = PlaneSlot(c, page, 0) + inPage; // of head 0; the next head's is a page of slots further
    const int pieces = c.KvHeads * LPH;
    const int4 *ks = reinterpret_cast<const int4 *>(p.KNew.Row(row)), *vs = reinterpret_cast<const int4 *>(p.VNew.Row(row));
    for (int i = lane; i < pieces; i += 128) {
        int4 a[4], b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (i + j * 32 < pieces) {
                a[j] = __ldg(ks + i + j * 32);
                b[j] = __ldg(vs + i + j * 32);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int x = i + j * 32;
            if (x < pieces) {
                const size_t at = (first + ((size_t)(x / LPH) << c.PageShift)) * LPH + x % LPH;
                reinterpret_cast<int4 *>(c.K)[at] = a[j];
                reinterpret_cast<int4 *>(c.V)[at] = b[j];
            }
        }
    }
    for (int h = lane; h < c.KvHeads; h += 32) {
        const size_t at = first + ((size_t)h << c.PageShift);
        const float sk = p.KScaleNew.Row(h)[row], sv = p.VScaleNew.Row(h)[row];
        if (SCALE_F16) {
            reinterpret_cast<__half *>(c.KScale)[at] = __float2half_rn(sk);
            reinterpret_cast<__half *>(c.VScale)[at] = __float2half_rn(sv);
        } else {
            reinterpret_cast<float *>(c.KScale)[at] = sk;
            reinterpret_cast<float *>(c.VScale)[at] = sv;
        }
        if (c.Pos) {
            c.Pos[at] = (p.Tokens ? p.Tokens[seq] : p.CtxLens[seq]) - back;
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

constexpr int SEL_THREADS = 512;
constexpr int SEL_WARPS = SEL_THREADS / 32;
constexpr int SEL_BINS = 2048;            // 11, 11 and 10 bits of the order
constexpr int SEL_MAX_CLUSTER = 8;
constexpr int SEL_SLOTS = 4096;           // slots of a CTA where there are CTAs enough
constexpr int SEL_MAX_SLICE = 48 * 1024;  // slots whose orders fit shared memory

// weights as unsigned integers of the same order; -0 counts as 0, NaN as the greatest; tokens that stay whatever their weight are above all
constexpr unsigned SEL_PINNED = 0xffffffffu, SEL_NAN = 0xfffffffeu;
__device__ __forceinline__ unsigned WeightOrder(float w)
{
    const unsigned b = __float_as_uint(w + 0.0f);
    return w != w ? SEL_NAN : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

// orders of slots slot .. slot + 3 (slot a multiple of 4); slots of pages outside the pool are the lightest
__device__ __forceinline__ uint4 SlotOrders(const TSelectParams &p, const int *table, int head, int slot, int newest, bool *bad)
{
    const TPages &c = p.C;
    const int page = table[slot >> c.PageShift];
    if ((unsigned)page >= (unsigned)c.PageCount) {
        *bad = true;
        return make_uint4(0, 0, 0, 0);
    }
    const size_t at = PlaneSlot(c, page, head) + (slot & ((1 << c.PageShift) - 1));
    const float4 w = *reinterpret_cast<const float4 *>(c.Weight + at);
    uint4 o = make_uint4(WeightOrder(w.x), WeightOrder(w.y), WeightOrder(w.z), WeightOrder(w.w));
    if (p.Recent > 0) {
        const int4 pos = c.Pos ? *reinterpret_cast<const int4 *>(c.Pos + at) : make_int4(slot, slot + 1, slot + 2, slot + 3);
        const int old = newest - p.Recent;
        o.x = pos.x > old ? SEL_PINNED : o.x;
        o.y = pos.y > old ? SEL_PINNED : o.y;
        o.z = pos.z > old ? SEL_PINNED : o.z;
        o.w = pos.w > old ? SEL_PINNED : o.w;
    }
    return o;
}

__device__ __forceinline__ uint4 ClusterLoad16(unsigned address)
{
    uint4 r;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(address) : "memory");
    return r;
}

struct TSelectShared {
    unsigned Hist[3][SEL_BINS];
    int WarpSum[SEL_WARPS];
    int Found[2];            // bin, and how many are still to be taken from it
    int4 Total;              // of this CTA: ties, holes, movers
    int4 WarpOf[SEL_WARPS];
};

// One cluster of CTAs per (sequence, key head); CTA `rank` has the slots [rank * slice, (rank + 1) * slice), each warp a contiguous run of
// them, four to a lane.  The keep-th largest order is found in three digits: counts of the digit among the orders that agree in the digits
// before (shared memory, the CTAs' counts added through distributed shared memory), then the sum from the top.  Ranks in slot order are
// ballots on top of the sums of the warps and CTAs before.  CACHED: the orders stay in shared memory after they are read once.
template <bool CACHED>
__global__ void __launch_bounds__(SEL_THREADS) PagedSelectKernel(const TSelectParams p)
{
    extern __shared__ uint4 cached[];
    __shared__ __align__(16) TSelectShared sh;
    const int head = blockIdx.x / p.Cluster, rank = blockIdx.x % p.Cluster, seq = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const TPages &c = p.C;
    for (int i = tid; i < 3 * SEL_BINS; i += SEL_THREADS) {
        sh.Hist[0][i] = 0;
    }
    PdlWait();
    PdlTrigger();
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
        for (int i = rank * SEL_THREADS + tid; i < p.MoveCap; i += p.Cluster * SEL_THREADS) {
            moves[i] = make_int2(-1, -1);
        }
        return;
    }
    const int *table = c.Table.Row(seq);
    const int newest = (p.Tokens ? p.Tokens[seq] : len) - 1;
    // slots of a CTA and of a warp: equal parts of what the sequence has, in whole steps of 128
    const int warps = p.Cluster * SEL_WARPS;
    const int per = ((len + warps - 1) / warps + 127) & ~127;
    const int slice = per * SEL_WARPS;
    const int beg = min(rank * slice + warp * per, len), end = min(beg + per, len);
    bool bad = false;
    auto orders = [&](int s) { return CACHED ? cached[(s - rank * slice) >> 2] : SlotOrders(p, table, head, s, newest, &bad); };
    auto count = [&](unsigned *hist, unsigned bin, bool in) {
        // equal bins of a whole warp (weights that are all zero) are one addition
        const unsigned first = __shfl_sync(0xffffffffu, bin, 0);
        if (__all_sync(0xffffffffu, in && bin == first)) {
            if (lane == 0) {
                atomicAdd(hist + bin, 32);
            }
        } else if (in) {
            atomicAdd(hist + bin, 1);
        }
    };
    __syncthreads(); // the counts are zero
#pragma unroll 2
    for (int s0 = beg; s0 < end; s0 += 128) {
        const int s = s0 + 4 * lane;
        uint4 o = make_uint4(0, 0, 0, 0);
        if (s < end) {
            o = SlotOrders(p, table, head, s, newest, &bad);
            if (CACHED) {
                cached[(s - rank * slice) >> 2] = o;
            }
        }
        count(sh.Hist[0], o.x >> 21, s < end);
        count(sh.Hist[0], o.y >> 21, s + 1 < end);
        count(sh.Hist[0], o.z >> 21, s + 2 < end);
        count(sh.Hist[0], o.w >> 21, s + 3 < end);
    }
    unsigned cut = 0;     // the digits found so far
    int take = p.Keep;    // how many of the orders that agree with them stay
#pragma unroll
    for (int digit = 0; digit < 3; ++digit) {
        constexpr int SHIFT[3] = {21, 10, 0};
        const int bits = digit == 2 ? 10 : 11;
        if (digit > 0) {
            const unsigned mask = digit == 1 ? 0xffe00000u : 0xfffffc00u;
            for (int s0 = beg; s0 < end; s0 += 128) {
                const int s = s0 + 4 * lane;
                const uint4 o = s < end ? orders(s) : make_uint4(0, 0, 0, 0);
                const unsigned low = (1u << bits) - 1;
                const bool x = s < end && (o.x & mask) == cut, y = s + 1 < end && (o.y & mask) == cut;
                const bool z = s + 2 < end && (o.z & mask) == cut, w = s + 3 < end && (o.w & mask) == cut;
                if (__any_sync(0xffffffffu, x | y | z | w)) {
                    count(sh.Hist[digit], o.x >> SHIFT[digit] & low, x);
                    count(sh.Hist[digit], o.y >> SHIFT[digit] & low, y);
                    count(sh.Hist[digit], o.z >> SHIFT[digit] & low, z);
                    count(sh.Hist[digit], o.w >> SHIFT[digit] & low, w);
                }
            }
        }
        if (p.Cluster > 1) {
            ClusterSync();
        } else {
            __syncthreads();
        }
        // thread t has bins [top - 4 t - 3, top - 4 t]: sums run from the largest bin down
        const int first = (1 << 11) - 4 - 4 * tid; // digits of 10 bits use the lower half, the rest is zero
        uint4 h = *reinterpret_cast<const uint4 *>(&sh.Hist[digit][first]);
        for (int r = 1; r < p.Cluster; ++r) {
            const uint4 o = ClusterLoad16(ClusterAddress(&sh.Hist[digit][first], (rank + r) % p.Cluster));
            h.x += o.x;
            h.y += o.y;
            h.z += o.z;
            h.w += o.w;
        }
        const int mine = (int)(h.x + h.y + h.z + h.w);
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            sum += lane >= o ? v : 0;
        }
        if (lane == 31) {
            sh.WarpSum[warp] = sum;
        }
        __syncthreads();
        for (int w = 0; w < warp; ++w) {
            sum += sh.WarpSum[w];
        }
        int above = sum - mine; // orders in larger bins
        if (above < take && sum >= take) {
            const unsigned b[4] = {h.w, h.z, h.y, h.x};
            int i = 0;
            while (above + (int)b[i] < take) {
                above += b[i++];
            }
            sh.Found[0] = first + 3 - i;
            sh.Found[1] = take - above;
            sh.Total.w = b[i]; // how many agree
        }
        __syncthreads();
        cut |= (unsigned)sh.Found[0] << SHIFT[digit];
        take = sh.Found[1];
    }
    // `take` of the orders equal to cut stay, the first ones in slot order; mostly that is all of them
    const bool allTies = sh.Total.w == take;
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
        int before = 0, total = 0;
        for (int w = 0; w < SEL_WARPS; ++w) {
            before += w < warp ? sh.WarpOf[w].x : 0;
            total += sh.WarpOf[w].x;
        }
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
    // two sweeps: count, then write
    int hole = 0, mover = 0, moved = 0;
#pragma unroll
    for (int sweep = 0; sweep < 2; ++sweep) {
        int left = ties;
        for (int s0 = beg; s0 < end; s0 += 128) {
            const int s = s0 + 4 * lane;
            const uint4 o4 = s < end ? orders(s) : make_uint4(0, 0, 0, 0);
            const unsigned o[4] = {o4.x, o4.y, o4.z, o4.w};
            const unsigned below = (1u << lane) - 1;
            bool keep[4];
            if (allTies) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    keep[i] = s + i < end && o[i] >= cut;
                }
            } else {
                unsigned tie[4];
                int before = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    tie[i] = __ballot_sync(0xffffffffu, s + i < end && o[i] == cut);
                    before += __popc(tie[i] & below);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool mine = tie[i] >> lane & 1;
                    keep[i] = s + i < end && (o[i] > cut || (mine && before < left));
                    before += mine;
                }
                left -= __popc(tie[0]) + __popc(tie[1]) + __popc(tie[2]) + __popc(tie[3]);
            }
            int hb = 0, mb = 0, hn = 0, mn = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned h = __ballot_sync(0xffffffffu, s + i < end && !keep[i] && s + i < p.Keep);
                const unsigned m = __ballot_sync(0xffffffffu, keep[i] && s + i >= p.Keep);
                hb += __popc(h & below);
                mb += __popc(m & below);
                hn += __popc(h);
                mn += __popc(m);
            }
            if (sweep) {
                int hr = hole + hb, mr = mover + mb;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (s + i < end && !keep[i] && s + i < p.Keep && hr < p.MoveCap) {
                        moves[hr++].x = s + i;
                    }
                    if (keep[i] && s + i >= p.Keep && mr < p.MoveCap) {
                        moves[mr++].y = s + i;
                    }
                }
            }
            hole += hn;
            mover += mn;
        }
        if (!sweep) {
            if (lane == 0) {
                sh.WarpOf[warp] = make_int4(0, hole, mover, 0);
            }
            __syncthreads();
            int4 total = make_int4(0, 0, 0, 0);
            hole = mover = 0;
            for (int w = 0; w < SEL_WARPS; ++w) {
                const int4 x = sh.WarpOf[w];
                hole += w < warp ? x.y : 0;
                mover += w < warp ? x.z : 0;
                total.y += x.y;
                total.z += x.z;
            }
            moved = total.z;
            if (p.Cluster > 1) {
                ClusterSync(); // the ties of Total have been read
                if (tid == 0) {
                    sh.Total = total;
                }
                ClusterSync();
                for (int r = 0; r < p.Cluster; ++r) {
                    const uint4 x = ClusterLoad16(ClusterAddress(&sh.Total, r));
                    hole += r < rank ? (int)x.y : 0;
                    mover += r < rank ? (int)x.z : 0;
                    moved += r != rank ? (int)x.z : 0;
                }
            }
            for (int i = moved + rank * SEL_THREADS + tid; i < p.MoveCap; i += p.Cluster * SEL_THREADS) {
                moves[i] = make_int2(-1, -1);
            }
            if (tid == 0 && rank == 0) {
                p.Counts[unit] = min(moved, p.MoveCap);
            }
        }
    }
    if (bad && p.Status) {
        atomicOr(p.Status, kDevBadSpan);
    }
    if (p.Cluster > 1) {
        ClusterSync(); // no CTA leaves while another reads its shared memory
    }
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
// carry a row of K and V.  Sources and destinations of a head are different slots (sources lie behind the budget), so no order is needed.
template <int D, int SCALE_BYTES>
__global__ void __launch_bounds__(MOV_WARPS * 32) PagedMoveKernel(const TMoveParams p)
{
    constexpr int LPM = 2 * D / 16, PER = 32 / LPM; // lanes per move, moves per step
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int head = blockIdx.y, seq = blockIdx.z;
    PdlTrigger();
    PdlWait();
    const TPages &c = p.C;
    const size_t unit = (size_t)seq * c.KvHeads + head;
    const int count = min(p.Counts[unit], p.MoveCap);
    const int base = (blockIdx.x * MOV_WARPS + warp) * 32;
    if (base >= count) {
        return;
    }
    const int2 *moves = p.Moves + unit * p.MoveCap;
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
            ok = pt >= 0 && pt < c.PageCount && pf >= 0 && pf < c.PageCount;
            if (ok) {
                to = PlaneSlot(c, pt, head) + (m.x & mask);
                of = PlaneSlot(c, pf, head) + (m.y & mask);
            }
        }
        if (!ok && p.Status) {
            atomicOr(p.Status, kDevBadSpan);
        }
    }
    const int n = min(32, count - base);
    const unsigned okMask = __ballot_sync(0xffffffffu, ok);
    const int sub = lane % LPM;
    const uint8_t *pool = sub < D / 16 ? c.K : c.V;
    const int piece = sub % (D / 16);
#pragma unroll 4
    for (int i = 0; i < 32; i += PER) {
        const int m = i + lane / LPM;
        const size_t t = __shfl_sync(0xffffffffu, to, m), f = __shfl_sync(0xffffffffu, of, m);
        if (m < n && (okMask >> m & 1)) {
            reinterpret_cast<int4 *>((uint8_t *)pool)[t * (D / 16) + piece] = reinterpret_cast<const int4 *>(pool)[f * (D / 16) + piece];
        }
    }
    if (ok) {
        if (SCALE_BYTES == 2) {
            const uint16_t a = reinterpret_cast<const uint16_t *>(c.KScale)[of], b = reinterpret_cast<const uint16_t *>(c.VScale)[of];
            reinterpret_cast<uint16_t *>(c.KScale)[to] = a;
            reinterpret_cast<uint16_t *>(c.VScale)[to] = b;
        } else {
            const uint32_t a = reinterpret_cast<const uint32_t *>(c.KScale)[of], b = reinterpret_cast<const uint32_t *>(c.VScale)[of];
            reinterpret_cast<uint32_t *>(c.KScale)[to] = a;
            reinterpret_cast<uint32_t *>(c.VScale)[to] = b;
        }
        if (c.Pos) {
            c.Pos[to] = c.Pos[of];
        }
        if (c.Weight) {
            c.Weight[to] = c.Weight[of];
        }
    }
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
    const bool f16 = cfg->scale_dtype == TSA_F16;
    const void *kern = cfg->head_dim == 128 ? (f16 ? (const void *)PagedAppendKernel<128, true> : (const void *)PagedAppendKernel<128, false>)
                                            : (f16 ? (const void *)PagedAppendKernel<64, true> : (const void *)PagedAppendKernel<64, false>);
    void *args[] = {&p};
    return CheckCuda(LaunchPdl(kern, dim3((rows + APP_WARPS - 1) / APP_WARPS), dim3(APP_WARPS * 32), 0, (cudaStream_t)stream, args), "tsa_paged_append launch");
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
    // CTAs of SEL_SLOTS slots while all of them are resident at once (four to an SM)
    p.Cluster = 1;
    while (p.Cluster < SEL_MAX_CLUSTER && longest > SEL_SLOTS * p.Cluster && 2ll * p.Cluster * kv->kv_heads * nSeq <= 4ll * sms) {
        p.Cluster *= 2;
    }
    const int warps = p.Cluster * SEL_WARPS;
    const int slice = ((longest + warps - 1) / warps + 127) / 128 * 128 * SEL_WARPS;
    const bool cached = slice <= SEL_MAX_SLICE;
    const void *kern = cached ? (const void *)PagedSelectKernel<true> : (const void *)PagedSelectKernel<false>;
    const size_t smem = cached ? (size_t)slice * sizeof(unsigned) : 0;
    if (smem > 16 * 1024) { // beyond 48 KB with the counts
        rc = CheckCuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SEL_MAX_SLICE * sizeof(unsigned)), "cudaFuncSetAttribute");
        if (rc != TSA_OK) {
            return rc;
        }
    }
    void *args[] = {&p};
    return CheckCuda(LaunchPdl(kern, dim3(kv->kv_heads * p.Cluster, nSeq), dim3(SEL_THREADS), smem, (cudaStream_t)stream, args, p.Cluster),
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
    TSA_REQUIRE(kv->kv_heads <= 65535, "tsa_paged_evict_move: %d key heads (at most 65535)", kv->kv_heads);
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

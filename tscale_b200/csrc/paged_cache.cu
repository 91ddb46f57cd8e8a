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
    int2 *Moves; // [nSeq][kvHeads][MoveCap]
    int *Counts; // [nSeq][kvHeads]
    int *NewLens;
    int *Status;
};

constexpr int SEL_THREADS = 1024;
constexpr int SEL_WARPS = SEL_THREADS / 32;

// weights as unsigned integers of the same order; -0 counts as 0, NaN as the greatest; tokens that stay whatever their weight are above all
constexpr unsigned SEL_PINNED = 0xffffffffu, SEL_NAN = 0xfffffffeu;
__device__ __forceinline__ unsigned WeightOrder(float w)
{
    const unsigned b = __float_as_uint(w + 0.0f);
    return w != w ? SEL_NAN : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ unsigned SlotOrder(const TSelectParams &p, const int *table, int head, int slot, int newest, int *bad)
{
    const TPages &c = p.C;
    const int page = table[slot >> c.PageShift];
    if (page < 0 || page >= c.PageCount) {
        *bad = 1;
        return 0;
    }
    const size_t at = PlaneSlot(c, page, head) + (slot & ((1 << c.PageShift) - 1));
    const int pos = c.Pos ? c.Pos[at] : slot;
    return pos > newest - p.Recent ? SEL_PINNED : WeightOrder(c.Weight[at]);
}

// sum over the block of each thread's value; every thread gets it
__device__ __forceinline__ int BlockSum(int v, int *red)
{
    v = __reduce_add_sync(0xffffffffu, v);
    __syncthreads(); // the previous sums have been read
    if ((threadIdx.x & 31) == 0) {
        red[threadIdx.x >> 5] = v;
    }
    __syncthreads();
    return __reduce_add_sync(0xffffffffu, red[threadIdx.x & 31]);
}

// One CTA per (sequence, key head).  Each warp owns a contiguous run of slots, so that ranks in slot order are a warp's ballots on top of
// the sums of the warps before it.  The keep-th largest weight is found bit by bit from the top (32 counts).
__global__ void __launch_bounds__(SEL_THREADS) PagedSelectKernel(const TSelectParams p)
{
    __shared__ int red[32];
    __shared__ int holesOf[32], moversOf[32], tiesOf[32];
    const int head = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    PdlTrigger();
    PdlWait();
    const TPages &c = p.C;
    const int len = p.CtxLens[seq];
    const size_t unit = (size_t)seq * c.KvHeads + head;
    int2 *moves = p.Moves + unit * p.MoveCap;
    const bool tooLong = len > p.MaxCtx || len > TableTokens(c);
    const bool none = len <= p.Keep || tooLong;
    if (tid == 0) {
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
    if (none) {
        for (int i = tid; i < p.MoveCap; i += SEL_THREADS) {
            moves[i] = make_int2(-1, -1);
        }
        return;
    }
    const int *table = c.Table.Row(seq);
    const int newest = (p.Tokens ? p.Tokens[seq] : len) - 1;
    const int per = ((len + SEL_WARPS - 1) / SEL_WARPS + 31) & ~31; // slots of a warp
    const int beg = min(warp * per, len), end = min(beg + per, len);
    int bad = 0;
    unsigned cut = 0; // largest value that at least Keep slots reach
    for (int bit = 31; bit >= 0; --bit) {
        const unsigned probe = cut | (1u << bit);
        int n = 0;
        for (int s = beg + lane; s < end; s += 32) {
            n += SlotOrder(p, table, head, s, newest, &bad) >= probe;
        }
        if (BlockSum(n, red) >= p.Keep) {
            cut = probe;
        }
    }
    int above = 0, equal = 0;
    for (int s = beg + lane; s < end; s += 32) {
        const unsigned o = SlotOrder(p, table, head, s, newest, &bad);
        above += o > cut;
        equal += o == cut;
    }
    equal = __reduce_add_sync(0xffffffffu, equal);
    if (lane == 0) {
        tiesOf[warp] = equal;
    }
    int take = p.Keep - BlockSum(above, red); // of the slots at the border, the first `take`
    for (int w = 0; w < warp; ++w) {
        take -= tiesOf[w];
    }
    // two sweeps: count, then write
    int hole = 0, mover = 0;
    for (int sweep = 0; sweep < 2; ++sweep) {
        int left = take;
        for (int s0 = beg; s0 < end; s0 += 32) {
            const int s = s0 + lane;
            const unsigned o = s < end ? SlotOrder(p, table, head, s, newest, &bad) : 0;
            const unsigned tie = __ballot_sync(0xffffffffu, s < end && o == cut);
            const bool kept = s < end && (o > cut || (o == cut && __popc(tie & ((1u << lane) - 1)) < left));
            left -= __popc(tie);
            const bool isHole = s < end && !kept && s < p.Keep, isMover = kept && s >= p.Keep;
            const unsigned hb = __ballot_sync(0xffffffffu, isHole), mb = __ballot_sync(0xffffffffu, isMover);
            if (sweep) {
                const int hr = hole + __popc(hb & ((1u << lane) - 1)), mr = mover + __popc(mb & ((1u << lane) - 1));
                if (isHole && hr < p.MoveCap) {
                    moves[hr].x = s;
                }
                if (isMover && mr < p.MoveCap) {
                    moves[mr].y = s;
                }
            }
            hole += __popc(hb);
            mover += __popc(mb);
        }
        if (!sweep) {
            if (lane == 0) {
                holesOf[warp] = hole;
                moversOf[warp] = mover;
            }
            __syncthreads();
            int total = 0;
            hole = mover = 0;
            for (int w = 0; w < SEL_WARPS; ++w) {
                hole += w < warp ? holesOf[w] : 0;
                mover += w < warp ? moversOf[w] : 0;
                total += moversOf[w];
            }
            for (int i = total + tid; i < p.MoveCap; i += SEL_THREADS) {
                moves[i] = make_int2(-1, -1);
            }
            if (tid == 0) {
                p.Counts[unit] = min(total, p.MoveCap);
            }
        }
    }
    if (bad && p.Status) {
        atomicOr(p.Status, kDevBadSpan);
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
    void *args[] = {&p};
    return CheckCuda(LaunchPdl((const void *)PagedSelectKernel, dim3(kv->kv_heads, nSeq), dim3(SEL_THREADS), 0, (cudaStream_t)stream, args),
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

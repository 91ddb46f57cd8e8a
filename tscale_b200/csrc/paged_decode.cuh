// Parameters and the division of the work of the attention over pages (paged_decode.cu, paged_decode_sm100.cu).
#pragma once
#include "paged.cuh"

namespace tsa {

constexpr int PD_ROWS = 16;         // query heads of a unit at most
constexpr int PD_MAX_CTAS = 1024;   // ranges that the partial sums have room for
constexpr int PD_RANGE_TILE = 128;  // slots of a tile of the ranges
constexpr int PD_UNIT_TILES = 2;    // tiles that beginning and ending a unit takes as long as
constexpr float PD_NO_REF = -1e30f; // reference of sums that have no key yet

// One unit = the query heads (at most 16) that share a key head of a sequence; key heads with more have several units.
struct TPagedDecodeParams {
    TPages C;
    const int *CtxLens, *Tokens;
    int NSeq, HeadCount, Group, HeadChunks; // HeadChunks: units per key head
    int Rows;                               // query heads of a unit's partial record
    int Cluster;                            // CTAs of a unit, where a cluster has it
    int MaxCtx, Window, OutDtype;
    bool ScaleF16;
    float Slope, DotScale, QVecScale;
    P2D<uint8_t> Q;
    P2D<float> QScale;
    P2D<char> Out;
    float *Partial;  // [CTA + unit][Rows][D + 4]: sums, reference, weight sum
    float *Lse;      // [nSeq][heads]: log2 of the weights' sum and the sink (caches that keep weights)
    float *Logits;   // [nSeq][heads][LogitRow]
    int LogitRow;
    int ListCap;     // keys that a CTA lists, where the kernel does
    int *Status;
};

__device__ __forceinline__ float Exp2(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float Log2(float x)
{
    float r;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// How far the logit of a key may lie above the reference: 2^(z - ref) * vScale stays within 2^headroom.  Value scales below 2^-80, zero among them,
// count as that here: weights then stay within 2^(80 + headroom), and the sum of 2^30 of them within float32.
__device__ __forceinline__ float ReferenceEdge(float vScale, float headroom)
{
    return headroom - fmaxf(Log2(fabsf(vScale)), -80.0f);
}

// tiles [First, First + Count) of TILE slots that hold the keys of a sequence; keys are slots [Beg, End) (of a cache with positions, some of
// them).  None where the sequence is longer than the call's bound or its row of the page table.
struct TSeqKeys {
    int First, Count, Beg, End;
};
template <int TILE>
__device__ __forceinline__ TSeqKeys SeqTiles(const TPagedDecodeParams &p, int s)
{
    const int len = p.CtxLens[s];
    TSeqKeys r = {0, 0, 0, 0};
    if (len <= 0 || len > p.MaxCtx || len > TableTokens(p.C)) {
        return r;
    }
    r.End = len;
    if (!p.C.Pos) {
        const int cur = len - 1;
        r.Beg = p.Window == 0 ? cur : max(0, cur - p.Window);
        r.End = p.Window == 0 ? len : cur;
    }
    r.First = r.Beg / TILE;
    r.Count = r.End > r.Beg ? (r.End + TILE - 1) / TILE - r.First : 0;
    return r;
}

// places of a unit in the row of all: PD_UNIT_TILES in front that stand for what it takes beside its tiles, then the tiles (ranges of equally
// many tiles: 49 us instead of 31 for 42 sequences of 40 .. 2523 slots, 12 key heads x 64, where some ranges had a dozen units of one tile)
__device__ __forceinline__ unsigned UnitPlaces(const TSeqKeys &keys)
{
    return keys.Count > 0 ? keys.Count + PD_UNIT_TILES : 0;
}

// A range's places: those of all units in a row (sequence by sequence, unit by unit) are cut into `ctas` equal ranges
__device__ __forceinline__ unsigned RangePlaces(unsigned total, unsigned ctas)
{
    return (total + ctas - 1) / ctas;
}

// the part of one unit that a range holds
struct TSegment {
    TSeqKeys Keys;
    int Seq, Unit; // Unit: of the sequence
    int TileBeg, TileEnd;
    bool Whole;    // all of the unit
};

// The segments of a range.  A whole warp calls these; every lane has the same answers.
struct TRangeWalk {
    unsigned At, End, SeqBase, Per;
    int Seq, UnitsPerSeq;

    // false: the range has no tiles; report: sequences that do not fit set the status word
    __device__ __forceinline__ bool Begin(const TPagedDecodeParams &p, int lane, unsigned cta, unsigned ctas, bool report)
    {
        UnitsPerSeq = p.C.KvHeads * p.HeadChunks;
        unsigned sum = 0;
        for (int s = lane; s < p.NSeq; s += 32) {
            sum += UnitPlaces(SeqTiles<PD_RANGE_TILE>(p, s));
            if (report && p.Status && (p.CtxLens[s] > p.MaxCtx || p.CtxLens[s] > TableTokens(p.C))) {
                atomicOr(p.Status, kDevBadSpan);
            }
        }
        const unsigned total = __reduce_add_sync(0xffffffffu, sum) * UnitsPerSeq;
        Per = RangePlaces(total, ctas);
        At = cta * Per;
        End = min(At + Per, total);
        if (At >= End) {
            return false;
        }
        unsigned before = 0;
        for (int s0 = 0;; s0 += 32) {
            const unsigned mine = s0 + lane < p.NSeq ? UnitPlaces(SeqTiles<PD_RANGE_TILE>(p, s0 + lane)) * UnitsPerSeq : 0;
            unsigned upTo = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned v = __shfl_up_sync(0xffffffffu, upTo, o);
                upTo += lane >= o ? v : 0;
            }
            const unsigned in = __ballot_sync(0xffffffffu, before + upTo > At);
            if (in) { // At < total: some sequence has it
                const int l = __ffs(in) - 1;
                SeqBase = before + __shfl_sync(0xffffffffu, upTo - mine, l);
                Seq = s0 + l;
                return ToTile(UnitPlaces(SeqTiles<PD_RANGE_TILE>(p, Seq)));
            }
            before += __shfl_sync(0xffffffffu, upTo, 31);
        }
    }
    // from a place in front of a unit's tiles to the first of them; false: the range ends before
    __device__ __forceinline__ bool ToTile(unsigned places)
    {
        const unsigned in = (At - SeqBase) % places;
        At += in < PD_UNIT_TILES ? PD_UNIT_TILES - in : 0;
        return At < End;
    }
    __device__ __forceinline__ TSegment Segment(const TPagedDecodeParams &p) const
    {
        TSegment r;
        r.Keys = SeqTiles<PD_RANGE_TILE>(p, Seq);
        r.Seq = Seq;
        const unsigned places = UnitPlaces(r.Keys);
        r.Unit = (int)((At - SeqBase) / places);
        const unsigned unitBeg = SeqBase + (unsigned)r.Unit * places + PD_UNIT_TILES;
        r.TileBeg = r.Keys.First + (int)(At - unitBeg);
        r.TileEnd = r.Keys.First + (int)(min(End, unitBeg + r.Keys.Count) - unitBeg);
        r.Whole = r.TileEnd - r.TileBeg == r.Keys.Count;
        return r;
    }
    // behind a segment; false: no more tiles
    __device__ __forceinline__ bool Next(const TPagedDecodeParams &p, const TSegment &seg)
    {
        At += seg.TileEnd - seg.TileBeg;
        if (At >= End) {
            return false;
        }
        unsigned places = UnitPlaces(seg.Keys);
        if (At == SeqBase + places * UnitsPerSeq) {
            SeqBase = At;
            do { // At < End: a later sequence has tiles
                places = UnitPlaces(SeqTiles<PD_RANGE_TILE>(p, ++Seq));
            } while (places == 0);
        }
        return ToTile(places);
    }
};

// record of the partial sums of the unit that CTA `cta` leaves unfinished.  cta + unit grows from each record to the next.
__device__ __forceinline__ float *PartialRecord(const TPagedDecodeParams &p, int headDim, unsigned cta, int seq, int unit, int row)
{
    return p.Partial + ((size_t)(cta + seq * (p.C.KvHeads * p.HeadChunks) + unit) * p.Rows + row) * (headDim + 4);
}

// paged_decode_sm100.cu: the attention of all ranges.  ctas: how many there are.
int LaunchPagedRanges(const TPagedDecodeParams &p, const tsa_paged_kv *kv, int headDim, bool e4m3, long long tilesMax, unsigned *ctas, cudaStream_t stream);

} // namespace tsa

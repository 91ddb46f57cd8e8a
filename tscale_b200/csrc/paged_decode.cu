// Attention of one new token per sequence over the paged key-value cache (tsa_paged_decode).
//
//   z_j = <q, k_j> * qScale * kScale_j * attDotScale - slope * (cur - pos_j)      keys with cur - window <= pos_j <= cur - 1
//   out = sum_j 2^z_j * vScale_j * v_j / (1 + sum_j 2^z_j)                        (the 1: the sink of tsa_att_decode)
//   weight_j += sum over the heads that share the key head of 2^z_j / (1 + sum)   (caches that keep weights)
//
// The stream of the cache bounds it: 2 D bytes of codes and two scales per key and key head, each read once.  The products run on the
// warp's matrix instructions, scores = q K^T with the query heads of a key head as rows and result^T = V^T weights^T with them as columns,
// so that up to 16 heads share what was loaded.  Fragments come straight from global memory: the order of the keys in a tile of 16 and of
// the head's dimensions are free, and are taken such that every lane loads 16 bytes at a time (lane = 4 g + t), of
//   K: key 4 (g / 2) + 2 n + g % 2 for column g of score block n, dimensions 16 t .. 16 t + 15 (and 64 more)
//   V: keys 4 t .. 4 t + 3, dimensions D / 8 g .. D / 8 g + D / 8 - 1
// which leaves lane (g, t) with the scores of head g for keys 4 t .. 4 t + 3: the weights are the second product's B fragment as they are.
//
// Weights: 2^(z - ref) * vScale in two f16 parts (22 bits; 2^-25 of the largest at worst), ref being the running maximum of
// z + log2 |vScale|, raised when a tile exceeds it by 2^8.  int8 products are exact in int32; e4m3 codes are exact in f16 and their
// products are summed in f32.
//
// Work: all keys of all (sequence, key head) units in a row, cut into equal ranges, one for each CTA that can be resident; a unit that a
// range border cuts leaves partial sums, which a second kernel joins in the order of the ranges (no atomics: the same bits every time).
#include "paged.cuh"

namespace tsa {

constexpr int PD_WARPS = 4;
constexpr int PD_THREADS = PD_WARPS * 32;
constexpr int PD_TILE = 16;              // keys of a warp's tile
constexpr int PD_MIN_TILES = 8;          // a CTA's range is at least two tiles per warp
constexpr int PD_MAX_CTAS = 1024;
constexpr int PD_ROWS = 16;              // query heads of a unit
constexpr float PD_NO_REF = -1e30f;      // reference of sums that have no key yet

struct TPagedDecodeParams {
    TPages C;
    const int *CtxLens, *Tokens;
    int NSeq, HeadCount, Group, HeadChunks; // HeadChunks: units per key head (16 query heads each)
    int Rows;                               // query heads of a unit's partial record
    int MaxCtx, Window, OutDtype;
    float Slope, DotScale, QVecScale;
    P2D<uint8_t> Q;
    P2D<float> QScale;
    P2D<char> Out;
    float *Partial;  // [CTA + unit][Rows][D + 4]: sums, reference, weight sum
    float *Lse;      // [nSeq][heads]: log2 of the weights' sum and the sink (caches that keep weights)
    float *Logits;   // [nSeq][heads][LogitRow]
    int LogitRow;
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
__device__ __forceinline__ uint4 LoadStream(const void *p)
{
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}
__device__ __forceinline__ uint2 LoadStream8(const void *p)
{
    uint2 r;
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
    return r;
}
__device__ __forceinline__ void MmaS8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void MmaF16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t E4M3PairToF16(uint32_t pair)
{
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)pair));
    return r;
}
// two bytes of `codes` (int8 offset by 128), picked by sel, as f16: 1024 + byte has the byte in the low bits of its significand
__device__ __forceinline__ uint32_t OffsetI8ToF16(uint32_t codes, uint32_t sel)
{
    const uint32_t x = __byte_perm(codes, 0x64646464u, sel);
    __half2 h = *reinterpret_cast<const __half2 *>(&x);
    h = __hsub2(h, __half2half2(__ushort_as_half(0x6480))); // 1152
    return *reinterpret_cast<uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t PackHalf2(float a, float b)
{
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t *>(&h);
}
// what a pair rounded to f16 leaves over
__device__ __forceinline__ uint32_t PackRest(uint32_t hi, float a, float b)
{
    const float2 f = __half22float2(*reinterpret_cast<__half2 *>(&hi));
    return PackHalf2(a - f.x, b - f.y);
}

// tiles [first, first + count) of 16 slots that hold the keys of a sequence; keys [beg, end) are slots when the cache has no positions
struct TSeqKeys {
    int First, Count, Beg, End;
};
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
    r.First = r.Beg / PD_TILE;
    r.Count = r.End > r.Beg ? (r.End + PD_TILE - 1) / PD_TILE - r.First : 0;
    return r;
}

// sum of the tiles of all sequences, by one warp; reports sequences that do not fit
__device__ __forceinline__ int TotalTiles(const TPagedDecodeParams &p, int lane, bool report)
{
    int sum = 0;
    for (int s = lane; s < p.NSeq; s += 32) {
        sum += SeqTiles(p, s).Count;
        if (report && p.Status && (p.CtxLens[s] > p.MaxCtx || p.CtxLens[s] > TableTokens(p.C))) {
            atomicOr(p.Status, kDevBadSpan);
        }
    }
    return __reduce_add_sync(0xffffffffu, sum);
}

// the sequence that holds tile `at` of the row of all sequences' tiles, each `mult` times; *base: the tile where it begins
__device__ __forceinline__ int SeqOfTile(const TPagedDecodeParams &p, unsigned at, int mult, int lane, unsigned *base)
{
    unsigned before = 0;
    for (int s0 = 0; s0 < p.NSeq; s0 += 32) {
        const unsigned mine = s0 + lane < p.NSeq ? SeqTiles(p, s0 + lane).Count * mult : 0;
        unsigned sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned v = __shfl_up_sync(0xffffffffu, sum, o);
            sum += lane >= o ? v : 0;
        }
        const unsigned in = __ballot_sync(0xffffffffu, before + sum > at);
        if (in) {
            const int l = __ffs(in) - 1;
            *base = before + __shfl_sync(0xffffffffu, sum - mine, l);
            return s0 + l;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    return -1;
}

// tiles of a CTA's range
__device__ __forceinline__ unsigned RangeTiles(unsigned total, unsigned ctas)
{
    return max((total + ctas - 1) / ctas, (unsigned)PD_MIN_TILES);
}

template <bool F16>
struct TScales; // scales of four keys
template <>
struct TScales<true> {
    uint2 X;
    __device__ __forceinline__ void Load(const char *p, size_t at) { X = LoadStream8(p + at * 2); }
    __device__ __forceinline__ float Get(int i) const
    {
        const uint32_t w = i < 2 ? X.x : X.y;
        return __half2float(__ushort_as_half((unsigned short)(i & 1 ? w >> 16 : w & 0xffff)));
    }
};
template <>
struct TScales<false> {
    uint4 X;
    __device__ __forceinline__ void Load(const char *p, size_t at) { X = LoadStream(p + at * 4); }
    __device__ __forceinline__ float Get(int i) const { return __uint_as_float(i == 0 ? X.x : i == 1 ? X.y : i == 2 ? X.z : X.w); }
};

// WIDE: more than eight query heads share a key head (otherwise rows 8 .. 15 of the scores are unused, and half the sums).
// SINGLE: a CTA has one whole unit (short contexts): no ranges, no partial sums, no second kernel.
template <int D, bool E4M3, bool SCALE_F16, bool WIDE, bool TRACK, bool SINGLE>
__global__ void __launch_bounds__(PD_THREADS, WIDE ? (D == 128 ? 3 : 4) : (D == 128 ? 4 : 6)) PagedDecodeKernel(const TPagedDecodeParams p)
{
    constexpr int MT = D / 16;                      // row blocks of the output, 16 dimensions each
    constexpr int HALVES = WIDE ? 2 : 1;            // blocks of eight query heads
    constexpr int KS = E4M3 ? D / 16 : D / 32;      // steps of the score product
    constexpr int ROWS = WIDE ? 16 : 8;
    __shared__ float accOf[PD_WARPS][ROWS][D + 4]; // [.][.][16 j + 2 g + b] for dimension D / 8 g + 2 j + b: no two lanes of a store meet in a bank
    __shared__ float refOf[PD_WARPS][ROWS], sumOf[PD_WARPS][ROWS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const TPages &c = p.C;
    const int unitsPerSeq = c.KvHeads * p.HeadChunks;
    PdlWait();
    PdlTrigger();

    unsigned at, rangeEnd, per = 0;
    int seq;
    unsigned seqBase;
    if (SINGLE) {
        seq = blockIdx.x / unitsPerSeq;
        const int n = SeqTiles(p, seq).Count;
        seqBase = 0;
        at = (blockIdx.x % unitsPerSeq) * n;
        rangeEnd = at + n;
        if (tid == 0 && p.Status && (p.CtxLens[seq] > p.MaxCtx || p.CtxLens[seq] > TableTokens(c))) {
            atomicOr(p.Status, kDevBadSpan);
        }
    } else {
        const unsigned total = (unsigned)TotalTiles(p, lane, blockIdx.x == 0 && warp == 0) * unitsPerSeq;
        per = RangeTiles(total, gridDim.x);
        at = blockIdx.x * per;
        rangeEnd = min(at + per, total);
        if (at >= rangeEnd) {
            return;
        }
        seq = SeqOfTile(p, at, unitsPerSeq, lane, &seqBase);
    }
    bool badPage = false;
    // one turn per unit that the range touches
    do {
        const TSeqKeys keys = SeqTiles(p, seq);
        const int inSeq = SINGLE ? (int)(blockIdx.x % unitsPerSeq) : (int)((at - seqBase) / keys.Count);
        const int head = inSeq / p.HeadChunks, chunk = inSeq % p.HeadChunks;
        const unsigned unitBeg = seqBase + (unsigned)inSeq * keys.Count;
        const int segBeg = keys.First + (int)(at - unitBeg), segEnd = keys.First + (int)(min(rangeEnd, unitBeg + keys.Count) - unitBeg);
        const bool whole = segBeg == keys.First && segEnd == keys.First + keys.Count;
        const int firstHead = head * p.Group + chunk * PD_ROWS;
        const int rows = min(p.Group - chunk * PD_ROWS, PD_ROWS);
        const int cur = (p.Tokens ? p.Tokens[seq] : p.CtxLens[seq]) - 1;
        const int *table = c.Table.Row(seq);
        const int tileShift = c.PageShift - 4, tileMask = (1 << tileShift) - 1;

        // the query heads of this lane's rows, in the dimensions' order of the fragments
        uint32_t qa[KS][4];
        float mult[2] = {0, 0};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int r = g + 8 * half;
            const bool live = (half == 0 || WIDE) && r < rows;
            uint32_t w[D / 16];
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
                uint4 x = make_uint4(0, 0, 0, 0);
                if (live) {
                    x = *reinterpret_cast<const uint4 *>(p.Q.Row(seq) + (firstHead + r) * D + i * 64 + t * 16);
                }
                w[i * 4 + 0] = x.x;
                w[i * 4 + 1] = x.y;
                w[i * 4 + 2] = x.z;
                w[i * 4 + 3] = x.w;
            }
            if (live) {
                mult[half] = p.DotScale * (p.QScale.Valid() ? p.QScale.Row(seq)[firstHead + r] : p.QVecScale);
            }
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                qa[i][half] = E4M3 ? E4M3PairToF16(w[E4M3 ? i : 0] & 0xffff) : w[E4M3 ? 0 : 2 * i];
                qa[i][half + 2] = E4M3 ? E4M3PairToF16(w[E4M3 ? i : 0] >> 16) : w[E4M3 ? 0 : 2 * i + 1];
            }
        }

        // acc[half][j]: heads 8 half + 2 t, + 1 (columns) of dimensions D / 8 g + 2 j (rows g), + 1 (rows g + 8)
        float acc[HALVES][MT][4];
#pragma unroll
        for (int i = 0; i < HALVES * MT; ++i) {
            acc[i / MT][i % MT][0] = acc[i / MT][i % MT][1] = acc[i / MT][i % MT][2] = acc[i / MT][i % MT][3] = 0;
        }
        float ref[2] = {PD_NO_REF, PD_NO_REF}, sum[2] = {0, 0};

        uint4 kr[2][D / 64];
        uint4 vr[4]; // D = 64 uses the first halves
        TScales<SCALE_F16> ks, vs;
        int4 ps;
        bool pageOk = true;
        const int keyRow = 4 * (g >> 1) + (g & 1); // of score block 0
        auto pageOf = [&](int tile) { return tile < segEnd ? table[tile >> tileShift] : 0; };
        auto slotOf = [&](int tile, int page) {
            pageOk = (unsigned)page < (unsigned)c.PageCount;
            return PlaneSlot(c, pageOk ? page : 0, head) + ((tile & tileMask) << 4);
        };
        auto loadK = [&](size_t slot) {
#pragma unroll
            for (int n = 0; n < 2; ++n) {
#pragma unroll
                for (int i = 0; i < D / 64; ++i) {
                    kr[n][i] = LoadStream(c.K + (slot + keyRow + 2 * n) * D + i * 64 + t * 16);
                }
            }
            ks.Load(c.KScale, slot + 4 * t);
            if (c.Pos) {
                ps = *reinterpret_cast<const int4 *>(c.Pos + slot + 4 * t);
            }
        };
        auto loadV = [&](size_t slot) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint8_t *src = c.V + (slot + 4 * t + i) * D + g * (D / 8);
                if (D == 128) {
                    vr[i] = LoadStream(src);
                } else {
                    const uint2 x = LoadStream8(src);
                    vr[i].x = x.x;
                    vr[i].y = x.y;
                }
            }
            vs.Load(c.VScale, slot + 4 * t);
        };

        int tile = segBeg + warp;
        if (tile < segEnd) {
            size_t slot = slotOf(tile, pageOf(tile));
            bool okNow = pageOk;
            loadK(slot);
            loadV(slot);
            int pageNext = pageOf(tile + PD_WARPS);
            for (; tile < segEnd; tile += PD_WARPS) {
                const bool more = tile + PD_WARPS < segEnd;
                const size_t slotNext = more ? slotOf(tile + PD_WARPS, pageNext) : slot;
                const bool okNext = pageOk;
                pageNext = pageOf(tile + 2 * PD_WARPS);
                badPage |= !okNow;

                // scores of block n, columns 2 t and 2 t + 1: keys 4 t + 2 n and 4 t + 2 n + 1
                float z[2][4]; // [row half][key]
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    if (E4M3) {
                        float d[4] = {0, 0, 0, 0};
#pragma unroll
                        for (int i = 0; i < D / 64; ++i) {
                            const uint32_t w[4] = {kr[n][i].x, kr[n][i].y, kr[n][i].z, kr[n][i].w};
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const uint32_t(&a)[4] = qa[E4M3 ? i * 4 + j : 0];
                                MmaF16(d, a[0], a[1], a[2], a[3], E4M3PairToF16(w[j] & 0xffff), E4M3PairToF16(w[j] >> 16));
                            }
                        }
                        z[0][2 * n] = d[0];
                        z[0][2 * n + 1] = d[1];
                        z[1][2 * n] = d[2];
                        z[1][2 * n + 1] = d[3];
                    } else {
                        int d[4] = {0, 0, 0, 0};
#pragma unroll
                        for (int i = 0; i < D / 64; ++i) {
                            MmaS8(d, qa[E4M3 ? 0 : 2 * i], kr[n][i].x, kr[n][i].y);
                            MmaS8(d, qa[E4M3 ? 0 : 2 * i + 1], kr[n][i].z, kr[n][i].w);
                        }
                        z[0][2 * n] = (float)d[0];
                        z[0][2 * n + 1] = (float)d[1];
                        z[1][2 * n] = (float)d[2];
                        z[1][2 * n + 1] = (float)d[3];
                    }
                }
                float kScale[4], vScale[4], lv[4];
                const int key0 = tile * PD_TILE + 4 * t;
                const int place[4] = {c.Pos ? ps.x : key0, c.Pos ? ps.y : key0 + 1, c.Pos ? ps.z : key0 + 2, c.Pos ? ps.w : key0 + 3};
                // a tile in the middle of the range of a cache without positions has no masked key
                const bool plain = okNow && !c.Pos && tile * PD_TILE >= keys.Beg && (tile + 1) * PD_TILE <= keys.End;
                bool valid[4] = {true, true, true, true};
                if (!plain) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = key0 + i;
                        valid[i] = okNow && key >= keys.Beg && key < keys.End;
                        if (c.Pos) {
                            const int far = cur - place[i];
                            valid[i] = valid[i] && (p.Window == 0 ? far == 0 : far >= 1 && far <= p.Window);
                        }
                        if (E4M3 && !valid[i]) {
                            vr[i] = make_uint4(0, 0, 0, 0); // what is in the slot may be NaN
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    kScale[i] = ks.Get(i);
                    vScale[i] = valid[i] ? vs.Get(i) : 0.0f;
                    lv[i] = fmaxf(Log2(fabsf(vScale[i])), -100.0f);
                    const float bias = p.Slope * (float)(cur - place[i]);
#pragma unroll
                    for (int half = 0; half < HALVES; ++half) {
                        z[half][i] = valid[i] ? z[half][i] * kScale[i] * mult[half] - bias : -INFINITY;
                    }
                }
                if (TRACK) {
#pragma unroll
                    for (int half = 0; half < HALVES; ++half) {
                        if (g + 8 * half < rows) {
                            float *dst = p.Logits + ((size_t)seq * p.HeadCount + firstHead + g + 8 * half) * p.LogitRow + key0;
                            *reinterpret_cast<float4 *>(dst) = make_float4(z[half][0], z[half][1], z[half][2], z[half][3]);
                        }
                    }
                }
                if (more) {
                    loadK(slotNext);
                }
                // raise the references of rows whose weights would leave f16's range
                bool raise = false;
#pragma unroll
                for (int half = 0; half < HALVES; ++half) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        raise |= z[half][i] + lv[i] > ref[half] + 8.0f;
                    }
                }
                if (__any_sync(0xffffffffu, raise)) {
                    float f[2] = {1, 1};
#pragma unroll
                    for (int half = 0; half < HALVES; ++half) {
                        float m = ref[half];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            m = fmaxf(m, z[half][i] + lv[i]);
                        }
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                        f[half] = Exp2(ref[half] - m);
                        ref[half] = m;
                        sum[half] *= f[half];
                    }
#pragma unroll
                    for (int half = 0; half < HALVES; ++half) {
                        const float f0 = __shfl_sync(0xffffffffu, f[half], 8 * t), f1 = __shfl_sync(0xffffffffu, f[half], 8 * t + 4);
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            acc[half][i][0] *= f0;
                            acc[half][i][1] *= f1;
                            acc[half][i][2] *= f0;
                            acc[half][i][3] *= f1;
                        }
                    }
                }
                uint32_t hi[2][2], lo[2][2]; // [row half][keys 0, 1 / 2, 3]
#pragma unroll
                for (int half = 0; half < HALVES; ++half) {
                    float w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        w[i] = Exp2(z[half][i] - ref[half]);
                        sum[half] += w[i];
                        w[i] *= vScale[i];
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        hi[half][i] = PackHalf2(w[2 * i], w[2 * i + 1]);
                        lo[half][i] = PackRest(hi[half][i], w[2 * i], w[2 * i + 1]);
                    }
                }
                // four dimensions at a time: bytes of keys 0, 1 and of keys 2, 3 side by side, then f16
#pragma unroll
                for (int r = 0; r < D / 32; ++r) {
                    uint32_t x[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[i] = r == 0 ? vr[i].x : r == 1 ? vr[i].y : r == 2 ? vr[i].z : vr[i].w;
                        if (!E4M3) {
                            x[i] ^= 0x80808080u;
                        }
                    }
                    const uint32_t a01 = __byte_perm(x[0], x[1], 0x5140), b01 = __byte_perm(x[0], x[1], 0x7362);
                    const uint32_t a23 = __byte_perm(x[2], x[3], 0x5140), b23 = __byte_perm(x[2], x[3], 0x7362);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t s01 = j ? b01 : a01, s23 = j ? b23 : a23;
                        uint32_t a0, a1, a2, a3;
                        if (E4M3) {
                            a0 = E4M3PairToF16(s01 & 0xffff);
                            a1 = E4M3PairToF16(s01 >> 16);
                            a2 = E4M3PairToF16(s23 & 0xffff);
                            a3 = E4M3PairToF16(s23 >> 16);
                        } else {
                            a0 = OffsetI8ToF16(s01, 0x4140);
                            a1 = OffsetI8ToF16(s01, 0x4342);
                            a2 = OffsetI8ToF16(s23, 0x4140);
                            a3 = OffsetI8ToF16(s23, 0x4342);
                        }
#pragma unroll
                        for (int half = 0; half < HALVES; ++half) {
                            float(&o)[4] = acc[half][r * 2 + j];
                            MmaF16(o, a0, a1, a2, a3, hi[half][0], hi[half][1]);
                            MmaF16(o, a0, a1, a2, a3, lo[half][0], lo[half][1]);
                        }
                    }
                }
                if (more) {
                    loadV(slotNext);
                }
                slot = slotNext;
                okNow = okNext;
            }
        }

        // the warps' sums meet in shared memory
#pragma unroll
        for (int half = 0; half < HALVES; ++half) {
            sum[half] += __shfl_xor_sync(0xffffffffu, sum[half], 1);
            sum[half] += __shfl_xor_sync(0xffffffffu, sum[half], 2);
            if (t == 0) {
                refOf[warp][g + 8 * half] = ref[half];
                sumOf[warp][g + 8 * half] = sum[half];
            }
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int r = 8 * half + 2 * t + b;
                if (r < rows) {
#pragma unroll
                    for (int j = 0; j < MT; ++j) {
                        *reinterpret_cast<float2 *>(&accOf[warp][r][16 * j + 2 * g]) = make_float2(acc[half][j][b], acc[half][j][2 + b]);
                    }
                }
            }
        }
        __syncthreads();
        for (int x = tid; x < rows * D; x += PD_THREADS) {
            const int r = x / D, i = x % D;
            const int d = (i >> 1 & 7) * (D / 8) + 2 * (i >> 4) + (i & 1);
            float m = refOf[0][r];
#pragma unroll
            for (int w = 1; w < PD_WARPS; ++w) {
                m = fmaxf(m, refOf[w][r]);
            }
            float s = 0, a = 0;
#pragma unroll
            for (int w = 0; w < PD_WARPS; ++w) {
                const float f = Exp2(refOf[w][r] - m);
                s = fmaf(f, sumOf[w][r], s);
                a = fmaf(f, accOf[w][r][i], a);
            }
            if (whole) {
                // the sink: weight 1 at logit 0
                const float all = fmaxf(m, -60.0f), f = Exp2(m - all);
                s = fmaf(f, s, Exp2(-all));
                StoreFromFloat(p.Out.Row(seq), (firstHead + r) * D + d, p.OutDtype, a * f / s);
                if (TRACK && d == 0) {
                    p.Lse[(size_t)seq * p.HeadCount + firstHead + r] = all + Log2(s);
                }
            } else {
                float *dst = p.Partial + ((size_t)(blockIdx.x + seq * unitsPerSeq + inSeq) * p.Rows + r) * (D + 4);
                dst[d] = a;
                if (d == 0) {
                    dst[D] = m;
                    dst[D + 1] = s;
                }
            }
        }
        if (SINGLE) {
            break;
        }
        at = unitBeg + (segEnd - keys.First);
        if (at < rangeEnd) {
            __syncthreads(); // shared memory is free again
            if (at == seqBase + (unsigned)keys.Count * unitsPerSeq) {
                seqBase = at;
                do {
                    ++seq;
                } while (SeqTiles(p, seq).Count == 0);
            }
        }
    } while (at < rangeEnd);
    if (badPage && p.Status) {
        atomicOr(p.Status, kDevBadSpan);
    }
}

// where a sequence's tiles begin in the row of all, and how long the ranges are; by one warp
__device__ __forceinline__ void SeqStart(const TPagedDecodeParams &p, int seq, int lane, unsigned ctas, unsigned *start, unsigned *per)
{
    int before = 0, all = 0;
    for (int s = lane; s < p.NSeq; s += 32) {
        const int n = SeqTiles(p, s).Count;
        before += s < seq ? n : 0;
        all += n;
    }
    const int units = p.C.KvHeads * p.HeadChunks;
    *start = (unsigned)__reduce_add_sync(0xffffffffu, before) * units;
    *per = RangeTiles((unsigned)__reduce_add_sync(0xffffffffu, all) * units, ctas);
}

// Joins the partial sums of one (sequence, query head) in the order of the ranges, and adds the sink.  Heads that one range held are
// finished already; sequences without keys get zeros.
template <int D>
__global__ void __launch_bounds__(128) PagedJoinKernel(const TPagedDecodeParams p, unsigned ctas)
{
    constexpr int LPC = D / 4, GROUPS = 128 / LPC;
    __shared__ float redMax[4];
    __shared__ float sumL[GROUPS];
    __shared__ float4 sumAcc[GROUPS][LPC];
    const int head = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
    const int kvHead = head / p.Group, inGroup = head % p.Group, chunk = inGroup / PD_ROWS, row = inGroup % PD_ROWS;
    const int units = p.C.KvHeads * p.HeadChunks, inSeq = kvHead * p.HeadChunks + chunk;
    unsigned start, per;
    // the lengths were there before the kernel whose sums are joined began
    SeqStart(p, seq, lane, ctas, &start, &per);
    const int count = SeqTiles(p, seq).Count;
    PdlWait();
    PdlTrigger();
    if (count == 0) {
        if (tid < D) {
            StoreFromFloat(p.Out.Row(seq), head * D + tid, p.OutDtype, 0.0f);
        }
        if (p.Lse && tid == 0) {
            p.Lse[(size_t)seq * p.HeadCount + head] = 0.0f;
        }
        return;
    }
    start += (unsigned)inSeq * count;
    const unsigned c0 = start / per, c1 = (start + count - 1) / per;
    if (c0 == c1) {
        return;
    }
    const int chunks = c1 - c0 + 1;
    const size_t stride = (size_t)p.Rows * (D + 4);
    const float *base = p.Partial + (size_t)(c0 + seq * units + inSeq) * stride + (size_t)row * (D + 4);
    float m = -60.0f;
    for (int i = tid; i < chunks; i += 128) {
        m = fmaxf(m, base[i * stride + D]);
    }
    m = WarpMax(m);
    if (lane == 0) {
        redMax[tid >> 5] = m;
    }
    __syncthreads();
    m = fmaxf(fmaxf(redMax[0], redMax[1]), fmaxf(redMax[2], redMax[3]));
    const int group = tid / LPC, sub = tid % LPC;
    float l = 0;
    float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (int i = group; i < chunks; i += GROUPS) {
        const float *src = base + i * stride;
        const float2 ml = *reinterpret_cast<const float2 *>(src + D);
        const float4 v = *reinterpret_cast<const float4 *>(src + 4 * sub);
        const float f = Exp2(ml.x - m);
        l = fmaf(f, ml.y, l);
        acc.x = fmaf(f, v.x, acc.x);
        acc.y = fmaf(f, v.y, acc.y);
        acc.z = fmaf(f, v.z, acc.z);
        acc.w = fmaf(f, v.w, acc.w);
    }
    sumAcc[group][sub] = acc;
    if (sub == 0) {
        sumL[group] = l;
    }
    __syncthreads();
    if (tid < D) {
        l = Exp2(-m);
        float a = 0;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            l += sumL[i];
            a += reinterpret_cast<const float *>(sumAcc[i])[tid];
        }
        StoreFromFloat(p.Out.Row(seq), head * D + tid, p.OutDtype, a / l);
        if (p.Lse && tid == 0) {
            p.Lse[(size_t)seq * p.HeadCount + head] = m + Log2(l);
        }
    }
}

// weight[slot] += sum over the heads of a key head of 2^(z - lse): one thread per slot
__global__ void __launch_bounds__(256) PagedWeightKernel(const TPagedDecodeParams p)
{
    const int head = blockIdx.y, seq = blockIdx.z, slot = blockIdx.x * 256 + threadIdx.x;
    PdlWait();
    PdlTrigger();
    const TPages &c = p.C;
    const TSeqKeys keys = SeqTiles(p, seq);
    if (slot < keys.First * PD_TILE || slot >= keys.End || keys.Count == 0) {
        return;
    }
    const int page = c.Table.Row(seq)[slot >> c.PageShift];
    if ((unsigned)page >= (unsigned)c.PageCount) {
        return;
    }
    const float *lse = p.Lse + (size_t)seq * p.HeadCount + head * p.Group;
    const float *z = p.Logits + ((size_t)seq * p.HeadCount + head * p.Group) * p.LogitRow + slot;
    float w = 0;
    for (int i = 0; i < p.Group; ++i) {
        w += Exp2(z[(size_t)i * p.LogitRow] - lse[i]);
    }
    c.Weight[PlaneSlot(c, page, head) + (slot & ((1 << c.PageShift) - 1))] += w;
}

// parts of the workspace, in this order
struct TPagedWorkspace {
    size_t Partial, Lse, Logits, Bytes;
    int LogitRow;
};
static TPagedWorkspace PagedWorkspace(int headDim, int nSeq, int kvHeads, int headCount, int maxCtx, bool track)
{
    auto round = [](size_t x) { return (x + 255) / 256 * 256; };
    const int group = headCount / kvHeads, rows = group < PD_ROWS ? group : PD_ROWS;
    const size_t units = (size_t)nSeq * kvHeads * ((group + PD_ROWS - 1) / PD_ROWS);
    TPagedWorkspace w;
    w.LogitRow = (maxCtx + PD_TILE - 1) / PD_TILE * PD_TILE;
    w.Partial = 0;
    w.Lse = round((PD_MAX_CTAS + units) * rows * (headDim + 4) * sizeof(float));
    w.Logits = w.Lse + (track ? round((size_t)nSeq * headCount * sizeof(float)) : 0);
    w.Bytes = w.Logits + (track ? (size_t)nSeq * headCount * w.LogitRow * sizeof(float) : 0);
    return w;
}

typedef void (*TPagedDecodeFn)(const TPagedDecodeParams);
template <int D, bool E4M3, bool SCALE_F16, bool WIDE, bool TRACK>
static TPagedDecodeFn PickSingle(bool single)
{
    return single ? PagedDecodeKernel<D, E4M3, SCALE_F16, WIDE, TRACK, true> : PagedDecodeKernel<D, E4M3, SCALE_F16, WIDE, TRACK, false>;
}
template <int D, bool E4M3, bool SCALE_F16>
static TPagedDecodeFn PickWide(bool wide, bool track, bool single)
{
    return wide ? (track ? PickSingle<D, E4M3, SCALE_F16, true, true>(single) : PickSingle<D, E4M3, SCALE_F16, true, false>(single))
                : (track ? PickSingle<D, E4M3, SCALE_F16, false, true>(single) : PickSingle<D, E4M3, SCALE_F16, false, false>(single));
}
template <int D>
static TPagedDecodeFn PickTypes(bool e4m3, bool f16, bool wide, bool track, bool single)
{
    return e4m3 ? (f16 ? PickWide<D, true, true>(wide, track, single) : PickWide<D, true, false>(wide, track, single))
                : (f16 ? PickWide<D, false, true>(wide, track, single) : PickWide<D, false, false>(wide, track, single));
}

} // namespace tsa

using namespace tsa;

extern "C" __attribute__((visibility("default"))) size_t tsa_paged_decode_workspace_bytes(const tsa_paged_cfg *cfg, const tsa_paged_kv *kv, int nSeq, int headCount,
    int maxCtx)
{
    if (!cfg || !kv || nSeq <= 0 || kv->kv_heads <= 0 || headCount < kv->kv_heads || maxCtx < 0) {
        return 0;
    }
    return PagedWorkspace(cfg->head_dim, nSeq, kv->kv_heads, headCount, maxCtx, kv->weight != nullptr).Bytes;
}

extern "C" __attribute__((visibility("default"))) int tsa_paged_decode(const tsa_paged_cfg *cfg, const tsa_paged_kv *kv, tsa_ptr2d pageTable,
    const int *ctxLens, const int *tokens, int nSeq, int maxCtx, tsa_ptr2d q, tsa_ptr2d qScale, int window, float alibiSlope, tsa_ptr2d out, int headCount,
    void *workspace, size_t workspaceBytes, int *statusWord, tsa_stream_t stream)
{
    TPagedDecodeParams p;
    int rc = CheckPages("tsa_paged_decode", cfg, kv, pageTable, ctxLens, nSeq, true, &p.C);
    if (rc != TSA_OK) {
        return rc;
    }
    TSA_REQUIRE(cfg->out_dtype >= TSA_F16 && cfg->out_dtype <= TSA_F32, "tsa_paged_decode: out dtype must be f16, bf16 or f32");
    TSA_REQUIRE(headCount > 0 && headCount % kv->kv_heads == 0, "tsa_paged_decode: %d query heads do not share %d key heads evenly", headCount, kv->kv_heads);
    TSA_REQUIRE(maxCtx >= 0 && window >= 0, "tsa_paged_decode: negative maxCtx or window");
    TSA_REQUIRE((kv->pos == nullptr) == (tokens == nullptr), "tsa_paged_decode: positions and the sequences' token counts go together");
    if (nSeq == 0) {
        return TSA_OK;
    }
    const int D = cfg->head_dim;
    TSA_REQUIRE((long long)headCount * D <= 0x7fffffff, "tsa_paged_decode: %d query heads", headCount);
    const int rowSize = headCount * D;
    TSA_REQUIRE(q.data && out.data, "tsa_paged_decode: null q or out");
    TSA_REQUIRE(q.xsize >= rowSize && q.ysize >= nSeq && out.xsize >= rowSize && out.ysize >= nSeq, "tsa_paged_decode: q/out extents");
    TSA_REQUIRE((uintptr_t)q.data % 16 == 0 && q.stride_bytes % 16 == 0, "tsa_paged_decode: q must be 16-byte aligned");
    TSA_REQUIRE((uintptr_t)out.data % 16 == 0 && out.stride_bytes % 16 == 0, "tsa_paged_decode: out must be 16-byte aligned");
    if (qScale.data) {
        TSA_REQUIRE(qScale.xsize >= headCount && qScale.ysize >= nSeq, "tsa_paged_decode: qScale extents");
        TSA_REQUIRE((uintptr_t)qScale.data % 4 == 0 && qScale.stride_bytes % 4 == 0, "tsa_paged_decode: qScale must be 4-byte aligned");
    }
    p.Group = headCount / kv->kv_heads;
    p.HeadChunks = (p.Group + PD_ROWS - 1) / PD_ROWS;
    p.Rows = p.Group < PD_ROWS ? p.Group : PD_ROWS;
    const long long room = TableTokens(p.C);
    const int longest = room < maxCtx ? (int)room : maxCtx;
    // keys of a sequence that a call looks at
    const long long keysMax = p.C.Pos ? longest : window == 0 ? 1 : longest < window ? longest : window;
    const long long tilesMax = (keysMax + PD_TILE - 1) / PD_TILE + 1;
    const long long units = (long long)nSeq * kv->kv_heads * p.HeadChunks;
    TSA_REQUIRE(units * tilesMax < (1ll << 31), "tsa_paged_decode: %d sequences of %d tokens with %d query heads are too much for one call", nSeq, longest, headCount);
    const bool track = kv->weight != nullptr;
    const TPagedWorkspace ws = PagedWorkspace(D, nSeq, kv->kv_heads, headCount, maxCtx, track);
    TSA_REQUIRE(workspace && workspaceBytes >= ws.Bytes, "tsa_paged_decode: workspace of %zu bytes needed, %zu given", ws.Bytes, workspaceBytes);
    TSA_REQUIRE((uintptr_t)workspace % 16 == 0, "tsa_paged_decode: workspace must be 16-byte aligned");
    p.CtxLens = ctxLens;
    p.Tokens = tokens;
    p.NSeq = nSeq;
    p.HeadCount = headCount;
    p.MaxCtx = maxCtx;
    p.Window = window;
    p.OutDtype = cfg->out_dtype;
    p.Slope = alibiSlope;
    p.DotScale = HostAttDotScale(D);
    p.QVecScale = cfg->qk_vec_scale;
    p.Q = P2D<uint8_t>(q);
    p.QScale = P2D<float>(qScale);
    p.Out = P2D<char>(out);
    p.Partial = (float *)workspace;
    p.Lse = track ? (float *)((char *)workspace + ws.Lse) : nullptr;
    p.Logits = (float *)((char *)workspace + ws.Logits);
    p.LogitRow = ws.LogitRow;
    p.Status = statusWord;
    const bool single = tilesMax <= PD_MIN_TILES + 1;
    const bool wide = p.Group > 8, e4m3 = cfg->kv_dtype == TSA_E4M3, f16 = cfg->scale_dtype == TSA_F16;
    const void *kern = (const void *)(D == 128 ? PickTypes<128>(e4m3, f16, wide, track, single) : PickTypes<64>(e4m3, f16, wide, track, single));
    int dev = 0, sms = 0, perSm = 0;
    rc = CheckCuda(cudaGetDevice(&dev), "cudaGetDevice");
    if (rc == TSA_OK) {
        rc = CheckCuda(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev), "cudaDeviceGetAttribute");
    }
    if (rc == TSA_OK) {
        rc = CheckCuda(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&perSm, kern, PD_THREADS, 0), "cudaOccupancyMaxActiveBlocksPerMultiprocessor");
    }
    if (rc != TSA_OK) {
        return rc;
    }
    long long grid = units;
    if (!single) {
        const long long resident = (long long)sms * (perSm < 1 ? 1 : perSm);
        grid = (units * tilesMax + PD_MIN_TILES - 1) / PD_MIN_TILES;
        grid = grid < resident ? grid : resident;
        grid = grid < PD_MAX_CTAS ? grid : PD_MAX_CTAS;
    }
    cudaStream_t s = (cudaStream_t)stream;
    unsigned ctas = (unsigned)grid;
    void *args[] = {&p, &ctas};
    rc = CheckCuda(LaunchPdl(kern, dim3(ctas), dim3(PD_THREADS), 0, s, args), "tsa_paged_decode launch");
    if (rc == TSA_OK && !single) {
        const void *join = D == 128 ? (const void *)PagedJoinKernel<128> : (const void *)PagedJoinKernel<64>;
        rc = CheckCuda(LaunchPdl(join, dim3(headCount, nSeq), dim3(128), 0, s, args), "tsa_paged_decode join launch");
    }
    if (rc == TSA_OK && track && longest > 0) {
        rc = CheckCuda(LaunchPdl((const void *)PagedWeightKernel, dim3((longest + 255) / 256, kv->kv_heads, nSeq), dim3(256), 0, s, args),
            "tsa_paged_decode weights launch");
    }
    return rc;
}

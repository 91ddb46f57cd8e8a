// Attention of one new token per sequence over the paged key-value cache (tsa_paged_decode).
//
//   z_j = <q, k_j> * qScale * kScale_j * attDotScale - slope * (cur - pos_j)      keys with cur - window <= pos_j <= cur - 1
//   out = sum_j 2^z_j * vScale_j * v_j / (1 + sum_j 2^z_j)                        (the 1: the sink of tsa_att_decode)
//   weight_j += sum over the heads that share the key head of 2^z_j / (1 + sum)   (caches that keep weights)
//
// The stream of the cache bounds it: 2 D bytes of codes and two scales per key and key head, each read once; for short caches the latency
// of what depends on one another does.  Two forms:
//   clusters (here): a cluster of up to 8 CTAs has a unit (the up to 16 query heads that share a key head of a sequence) and joins its sums
//     through distributed shared memory: one kernel, for caches of up to 4080 slots while all clusters are resident at once, and for windows of
//     up to 1024 positions of longer caches with positions, whose keys it lists first.
//   ranges (paged_decode_sm100.cu): all keys of all units, in a row, are cut into equal ranges, one for each CTA that can be resident; a
//     unit that a range border cuts leaves partial sums, which a second kernel joins in the order of the ranges.
// No atomics in either: the same bits every time.  Measured: 12 heads x 64 of one sequence of 1000 slots 5.3 us (the host's call takes as long); 64
// key heads of 1024 slots, two query heads x 128 each, 7.4 us; and with the keys' weights, 4 key heads of 2049 slots, 7.8.
//
// Cluster form.  The products run on the warp's matrix instructions, scores = q K^T with the query heads as rows and result^T = V^T
// weights^T with them as columns.  Fragments come straight from global memory: the order of the keys in a tile of 16 and of the head's
// dimensions are free, and are taken such that every lane loads 16 bytes at a time (lane = 4 g + t), of
//   K: key 4 (g / 2) + 2 n + g % 2 for column g of score block n, dimensions 16 t .. 16 t + 15 (and 64 more)
//   V: keys 4 t .. 4 t + 3, dimensions D / 8 g .. D / 8 g + D / 8 - 1
// which leaves lane (g, t) with the scores of head g for keys 4 t .. 4 t + 3: the weights are the second product's B fragment as they are.
// Weights: 2^(z - ref) * vScale in two f16 parts (22 bits; 2^-25 of the largest at worst), ref being the running maximum of
// z + log2 |vScale|, raised when a tile exceeds it by 2^8.  int8 products are exact in int32; e4m3 codes are exact in f16 and their
// products are summed in f32.
#include "paged_decode.cuh"
#include <type_traits>

namespace tsa {

constexpr int PD_WARPS = 4;
constexpr int PD_ONE_WARP_TILES = 8;     // of a unit that one warp has, at most
constexpr int PD_TILE = 16;              // keys of a warp's tile
constexpr int PD_MIN_TILES = 8;          // of a CTA: two tiles per warp
constexpr int PD_MAX_CLUSTER = 8;
constexpr int PD_MAX_LIST = 1024;        // keys that a CTA lists
constexpr float PD_EDGE = 8.0f;          // log2 of the largest weight

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
__device__ __forceinline__ void LoadStream(const void *p, uint4 *r)
{
    *r = LoadStream(p);
}
__device__ __forceinline__ void LoadStream(const void *p, uint2 *r)
{
    *r = LoadStream8(p);
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

// scales of four keys
template <bool F16>
struct TScales;
template <>
struct TScales<true> {
    uint2 X;
    __device__ __forceinline__ void Load(const char *p, size_t at) { X = LoadStream8(p + at * 2); }
    __device__ __forceinline__ void Gather(const char *p, const size_t (&at)[4])
    {
        const unsigned short *s = reinterpret_cast<const unsigned short *>(p);
        const unsigned a = s[at[0]], b = s[at[1]], c = s[at[2]], d = s[at[3]];
        X = make_uint2(a | b << 16, c | d << 16);
    }
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
    __device__ __forceinline__ void Gather(const char *p, const size_t (&at)[4])
    {
        const unsigned *s = reinterpret_cast<const unsigned *>(p);
        X = make_uint4(s[at[0]], s[at[1]], s[at[2]], s[at[3]]);
    }
    __device__ __forceinline__ float Get(int i) const { return __uint_as_float(i == 0 ? X.x : i == 1 ? X.y : i == 2 ? X.z : X.w); }
};

__device__ __forceinline__ float ClusterLoad(const float *mine, int rank)
{
    float r;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(r) : "r"(ClusterAddress(mine, rank)) : "memory");
    return r;
}

// One cluster of p.Cluster CTAs per unit.  WIDE: more than eight query heads share a key head (otherwise rows 8 .. 15 of the scores are
// unused, and half the sums).  A warp works on U tiles of 16 keys at a time, 4 KB of K and V, and holds the loads of its next ones in
// registers meanwhile.
// SPARSE: of a cache with positions, whose tokens may be in any order, and a window much shorter than it.  The CTA looks at the positions of its
// slots first and lists those inside the window; its tiles are then 16 of the list each, gathered row by row.
// WARPS: four; one where there are many units of a few tiles.
template <int D, bool E4M3, bool SCALE_F16, bool WIDE, bool SPARSE, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, (WIDE ? 3 : 4) * (PD_WARPS / WARPS)) PagedClusterKernel(const TPagedDecodeParams p)
{
    constexpr int THREADS = WARPS * 32;
    constexpr int U = 128 / D, STEP = WARPS * U;
    constexpr int MT = D / 16;                      // row blocks of the output, 16 dimensions each
    constexpr int HALVES = WIDE ? 2 : 1;            // blocks of eight query heads
    constexpr int KS = E4M3 ? D / 16 : D / 32;      // steps of the score product
    constexpr int ROWS = 8 * HALVES;
    typedef typename std::conditional<D == 128, uint4, uint2>::type TPiece; // D / 8 dimensions of a key
    extern __shared__ __align__(16) float logits[]; // of this CTA's keys, [rows][p.LogitRow]
    // SPARSE, behind the logits: where the listed keys are in the planes, and how far from the query's position
    size_t *const listAt = reinterpret_cast<size_t *>(logits + (p.C.Weight ? p.Rows * p.LogitRow : 0));
    int *const listFar = reinterpret_cast<int *>(listAt + p.ListCap);
    __shared__ int listOf[WARPS];
    __shared__ __align__(16) float accOf[WARPS][ROWS][D + 4]; // [.][.][16 j + 2 g + b] for dimension D / 8 g + 2 j + b: no two lanes of a store meet in a bank
    __shared__ float refOf[WARPS][ROWS], sumOf[WARPS][ROWS], ctaRef[ROWS], ctaSum[ROWS], lseOf[ROWS], factorOf[ROWS][PD_MAX_CLUSTER];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const TPages &c = p.C;
    const int unitsPerSeq = c.KvHeads * p.HeadChunks, ctas = p.Cluster, rank = blockIdx.x % ctas, unit = blockIdx.x / ctas;
    const int seq = unit / unitsPerSeq, head = unit % unitsPerSeq / p.HeadChunks, chunk = unit % p.HeadChunks;
    const int firstHead = head * p.Group + chunk * PD_ROWS, rows = min(p.Group - chunk * PD_ROWS, PD_ROWS);
    PdlTrigger();
    PdlWait();
    if (tid == 0 && p.Status && (p.CtxLens[seq] > p.MaxCtx || p.CtxLens[seq] > TableTokens(c))) {
        atomicOr(p.Status, kDevBadSpan);
    }
    const TSeqKeys keys = SeqTiles<PD_TILE>(p, seq);
    const int per = (keys.Count + ctas - 1) / ctas;
    int segBeg = keys.First + min(rank * per, keys.Count), segEnd = min(segBeg + per, keys.First + keys.Count);
    const int cur = (p.Tokens ? p.Tokens[seq] : p.CtxLens[seq]) - 1;
    const int *table = c.Table.Row(seq);
    const int tileShift = c.PageShift - 4, tileMask = (1 << tileShift) - 1;
    // keys of this CTA; a key at distance cur - position is attended if (unsigned)(distance - nearest) < spread
    int keyBeg = keys.Beg, keyEnd = min(keys.End, segEnd * PD_TILE);
    const int nearest = p.Window > 0 ? 1 : 0;
    const unsigned spread = p.Window > 0 ? p.Window : 1;
    const bool track = c.Weight != nullptr;
    bool badPage = false;
    if (SPARSE) {
        // each warp has a contiguous part of the CTA's slots; it counts, then it lists them
        const int slots = ((keyEnd - segBeg * PD_TILE + WARPS - 1) / WARPS + 3) & ~3;
        const int beg = segBeg * PD_TILE + warp * slots, end = min(beg + slots, keyEnd);
        int at = 0;
        auto scan = [&](bool write) {
            constexpr int AHEAD = 4;
            for (int s0 = beg; s0 < end; s0 += 128 * AHEAD) {
                int page[AHEAD];
                int4 pos[AHEAD];
                size_t where[AHEAD];
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) {
                    const int s = s0 + 128 * j + 4 * lane;
                    page[j] = s < end ? table[s >> c.PageShift] : 0;
                    badPage |= (unsigned)page[j] >= (unsigned)c.PageCount;
                }
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) {
                    const int s = s0 + 128 * j + 4 * lane;
                    where[j] = PlaneSlot(c, (unsigned)page[j] < (unsigned)c.PageCount ? page[j] : 0, head) + (s & ((1 << c.PageShift) - 1));
                    pos[j] = *reinterpret_cast<const int4 *>(c.Pos + where[j]);
                }
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) {
                    const int s = s0 + 128 * j + 4 * lane, far[4] = {cur - pos[j].x, cur - pos[j].y, cur - pos[j].z, cur - pos[j].w};
                    unsigned in = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        in |= (unsigned)(s + i < end && (unsigned)page[j] < (unsigned)c.PageCount && (unsigned)(far[i] - nearest) < spread) << i;
                    }
                    if (!__any_sync(0xffffffffu, in)) {
                        continue;
                    }
                    int before = __popc(in);
                    const int mine = before;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int v = __shfl_up_sync(0xffffffffu, before, o);
                        before += lane >= o ? v : 0;
                    }
                    if (write) {
                        int to = at + before - mine;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (in >> i & 1) {
                                if (to < p.ListCap) {
                                    listAt[to] = where[j] + i;
                                    listFar[to] = far[i];
                                }
                                ++to;
                            }
                        }
                    }
                    at += __shfl_sync(0xffffffffu, before, 31);
                }
            }
        };
        scan(false);
        if (lane == 0) {
            listOf[warp] = at;
        }
        __syncthreads();
        at = 0;
        keyEnd = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            at += w < warp ? listOf[w] : 0;
            keyEnd += listOf[w];
        }
        scan(true);
        __syncthreads();
        // from here on, keys are places of the list.  It has room for a key at each position of the window; where positions repeat, for no more
        if (keyEnd > p.ListCap && tid == 0 && p.Status) {
            atomicOr(p.Status, kDevBadSpan);
        }
        keyEnd = min(keyEnd, p.ListCap);
        keyBeg = segBeg = 0;
        segEnd = (keyEnd + PD_TILE - 1) / PD_TILE;
    }

    // the query heads of this lane's rows, in the dimensions' order of the fragments
    uint32_t qa[KS][4];
    float mult[2] = {0, 0};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int r = g + 8 * half;
        const bool live = half < HALVES && r < rows;
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
    float ref[HALVES], sum[HALVES];
#pragma unroll
    for (int half = 0; half < HALVES; ++half) {
        ref[half] = PD_NO_REF;
        sum[half] = 0;
    }

    uint4 kr[U][2][D / 64];
    TPiece vr[U][4];
    TScales<SCALE_F16> ks[U], vs[U];
    int4 ps[U];
    const int keyRow = 4 * (g >> 1) + (g & 1); // of score block 0
    const size_t kLane = (size_t)keyRow * D + t * 16, vLane = (size_t)(4 * t) * D + g * (D / 8);
    auto pageOf = [&](int tile) { return SPARSE ? 0 : tile < segEnd ? table[tile >> tileShift] : -1; };
    auto listed = [&](size_t i) { return listAt[min((int)i, keyEnd - 1)]; };
    // the slots of a tile; a tile that there is not, or whose page is outside the pool, reads page 0 and is masked
    auto slotOf = [&](int tile, int page) {
        return SPARSE ? (size_t)tile * PD_TILE : PlaneSlot(c, (unsigned)page < (unsigned)c.PageCount ? page : 0, head) + ((tile & tileMask) << 4);
    };
    auto loadK = [&](const size_t (&slot)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint8_t *src = c.K + slot[u] * D + kLane;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const uint8_t *row = SPARSE ? c.K + listed(slot[u] + keyRow + 2 * n) * D + t * 16 : src + 2 * n * D;
#pragma unroll
                for (int i = 0; i < D / 64; ++i) {
                    kr[u][n][i] = LoadStream(row + i * 64);
                }
            }
            if (SPARSE) {
                const size_t at[4] = {listed(slot[u] + 4 * t), listed(slot[u] + 4 * t + 1), listed(slot[u] + 4 * t + 2), listed(slot[u] + 4 * t + 3)};
                ks[u].Gather(c.KScale, at);
                vs[u].Gather(c.VScale, at);
                continue;
            }
            ks[u].Load(c.KScale, slot[u] + 4 * t);
            vs[u].Load(c.VScale, slot[u] + 4 * t); // with K: the weights need it before V
            if (c.Pos) {
                ps[u] = *reinterpret_cast<const int4 *>(c.Pos + slot[u] + 4 * t);
            }
        }
    };
    auto loadV = [&](const size_t (&slot)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint8_t *src = c.V + slot[u] * D + vLane;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                LoadStream(SPARSE ? c.V + listed(slot[u] + 4 * t + i) * D + g * (D / 8) : src + i * D, &vr[u][i]);
            }
        }
    };

    int tile = segBeg + warp * U;
    if (tile < segEnd) {
        size_t slot[U];
        int page[U];
        bool ok[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            page[u] = pageOf(tile + u);
            slot[u] = slotOf(tile + u, page[u]);
            ok[u] = (unsigned)page[u] < (unsigned)c.PageCount;
            badPage |= !ok[u] && tile + u < segEnd;
        }
        loadK(slot);
        loadV(slot);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            page[u] = pageOf(tile + STEP + u);
        }
        for (; tile < segEnd; tile += STEP) {
            const bool more = tile + STEP < segEnd;
            bool okNow[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                okNow[u] = ok[u];
                if (more) {
                    slot[u] = slotOf(tile + STEP + u, page[u]);
                    ok[u] = (unsigned)page[u] < (unsigned)c.PageCount;
                    badPage |= !ok[u] && tile + STEP + u < segEnd;
                }
                page[u] = pageOf(tile + 2 * STEP + u);
            }

            // scores of block n, columns 2 t and 2 t + 1: keys 4 t + 2 n and 4 t + 2 n + 1; then logits
            float z[U][HALVES][4], vScale[U][4], edge[U][4];
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    float dot[4];
                    if (E4M3) {
                        float d[4] = {0, 0, 0, 0};
#pragma unroll
                        for (int i = 0; i < KS; ++i) {
                            const uint32_t w = reinterpret_cast<const uint32_t *>(&kr[u][n][E4M3 ? i / 4 : 0])[i % 4];
                            MmaF16(d, qa[i][0], qa[i][1], qa[i][2], qa[i][3], E4M3PairToF16(w & 0xffff), E4M3PairToF16(w >> 16));
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            dot[i] = d[i];
                        }
                    } else {
                        int d[4] = {0, 0, 0, 0};
#pragma unroll
                        for (int i = 0; i < KS; ++i) {
                            const uint4 &k4 = kr[u][n][E4M3 ? 0 : i / 2];
                            MmaS8(d, qa[i], i % 2 ? k4.z : k4.x, i % 2 ? k4.w : k4.y);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            dot[i] = (float)d[i];
                        }
                    }
#pragma unroll
                    for (int half = 0; half < HALVES; ++half) {
                        z[u][half][2 * n] = dot[2 * half];
                        z[u][half][2 * n + 1] = dot[2 * half + 1];
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int key0 = (tile + u) * PD_TILE + 4 * t;
                int far[4] = {cur - key0, cur - key0 - 1, cur - key0 - 2, cur - key0 - 3};
                if (SPARSE) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        far[i] = listFar[min(key0 + i, keyEnd - 1)];
                    }
                } else if (c.Pos) {
                    far[0] = cur - ps[u].x;
                    far[1] = cur - ps[u].y;
                    far[2] = cur - ps[u].z;
                    far[3] = cur - ps[u].w;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    vScale[u][i] = vs[u].Get(i);
                    const float kScale = ks[u].Get(i);
#pragma unroll
                    for (int half = 0; half < HALVES; ++half) {
                        z[u][half][i] *= kScale * mult[half];
                    }
                }
                if (p.Slope != 0) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
#pragma unroll
                        for (int half = 0; half < HALVES; ++half) {
                            z[u][half][i] = fmaf(-p.Slope, (float)far[i], z[u][half][i]);
                        }
                    }
                }
                // a tile in the middle of the range of a cache without positions has no masked key
                if (!okNow[u] || (!SPARSE && c.Pos) || (tile + u) * PD_TILE < keyBeg || (tile + u + 1) * PD_TILE > keyEnd) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool valid = okNow[u] && key0 + i >= keyBeg && key0 + i < keyEnd && (unsigned)(far[i] - nearest) < spread;
                        if (!valid) { // what is in the slot may be NaN
                            vScale[u][i] = 0;
                            if (E4M3) {
                                vr[u][i] = TPiece{};
                            }
#pragma unroll
                            for (int half = 0; half < HALVES; ++half) {
                                z[u][half][i] = -INFINITY;
                            }
                        }
                    }
                }
                if (track && tile + u < segEnd) {
#pragma unroll
                    for (int half = 0; half < HALVES; ++half) {
                        if (g + 8 * half < rows) {
                            *reinterpret_cast<float4 *>(logits + (g + 8 * half) * p.LogitRow + key0 - segBeg * PD_TILE) =
                                make_float4(z[u][half][0], z[u][half][1], z[u][half][2], z[u][half][3]);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    edge[u][i] = ReferenceEdge(vScale[u][i], PD_EDGE);
                }
            }
            if (more) {
                loadK(slot);
            }
            // raise the references of rows whose weights would leave f16's range
            bool raise = false;
#pragma unroll
            for (int i = 0; i < U * HALVES * 4; ++i) {
                raise |= z[i / 4 / HALVES][i / 4 % HALVES][i % 4] - ref[i / 4 % HALVES] > edge[i / 4 / HALVES][i % 4];
            }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int half = 0; half < HALVES; ++half) {
                    float m = ref[half];
#pragma unroll
                    for (int i = 0; i < U * 4; ++i) {
                        m = fmaxf(m, z[i / 4][half][i % 4] - edge[i / 4][i % 4] + PD_EDGE);
                    }
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                    const float f = Exp2(ref[half] - m);
                    ref[half] = m;
                    sum[half] *= f;
                    const float f0 = __shfl_sync(0xffffffffu, f, 8 * t), f1 = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        acc[half][i][0] *= f0;
                        acc[half][i][1] *= f1;
                        acc[half][i][2] *= f0;
                        acc[half][i][3] *= f1;
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                uint32_t hi[HALVES][2], lo[HALVES][2]; // [.][keys 0, 1 / 2, 3]
#pragma unroll
                for (int half = 0; half < HALVES; ++half) {
                    float w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        w[i] = Exp2(z[u][half][i] - ref[half]);
                        sum[half] += w[i];
                        w[i] *= vScale[u][i];
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
                        x[i] = reinterpret_cast<const uint32_t *>(&vr[u][i])[r];
                        if (!E4M3) {
                            x[i] ^= 0x80808080u;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t s01 = __byte_perm(x[0], x[1], j ? 0x7362 : 0x5140), s23 = __byte_perm(x[2], x[3], j ? 0x7362 : 0x5140);
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
            }
            if (more) {
                loadV(slot);
            }
        }
    }
    if (badPage && p.Status) {
        atomicOr(p.Status, kDevBadSpan);
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
    // this CTA's keys' weights so far are on their way while the sums are joined
    constexpr int OWN_KEYS = (SPARSE ? PD_MAX_LIST : WARPS == 1 ? PD_ONE_WARP_TILES * PD_TILE : 4 * PD_MIN_TILES * PD_TILE) / THREADS; // of a thread at most
    constexpr size_t NOWHERE = ~(size_t)0;
    const int keyFirst = max(keyBeg, segBeg * PD_TILE);
    size_t slotAt[OWN_KEYS];
    float before[OWN_KEYS];
    if (track) {
#pragma unroll
        for (int i = 0; i < OWN_KEYS; ++i) {
            const int key = keyFirst + i * THREADS + tid;
            if (SPARSE) {
                slotAt[i] = key < keyEnd ? listAt[key] : NOWHERE;
            } else {
                const int page = key < keyEnd ? table[key >> c.PageShift] : -1;
                slotAt[i] = (unsigned)page < (unsigned)c.PageCount ? PlaneSlot(c, page, head) + (key & ((1 << c.PageShift) - 1)) : NOWHERE;
            }
            before[i] = slotAt[i] != NOWHERE ? c.Weight[slotAt[i]] : 0.0f;
        }
    }
    __syncthreads();
    // the CTA's sums: in the place of its first warp's
    for (int x = tid; x < rows * D; x += THREADS) {
        const int r = x / D, i = x % D;
        float m = refOf[0][r];
#pragma unroll
        for (int w = 1; w < WARPS; ++w) {
            m = fmaxf(m, refOf[w][r]);
        }
        float a = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            a = fmaf(Exp2(refOf[w][r] - m), accOf[w][r][i], a);
        }
        accOf[0][r][i] = a;
    }
    if (tid < rows) {
        float m = refOf[0][tid], s = 0;
#pragma unroll
        for (int w = 1; w < WARPS; ++w) {
            m = fmaxf(m, refOf[w][tid]);
        }
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            s = fmaf(Exp2(refOf[w][tid] - m), sumOf[w][tid], s);
        }
        ctaRef[tid] = m;
        ctaSum[tid] = s;
    }
    if (ctas > 1) {
        ClusterSync();
    } else {
        __syncthreads();
    }
    // every CTA of the cluster finishes a part of the result from all their sums: eight threads per row find the factors of the CTAs' sums.
    // The reference is at least -60: the sink, weight 1 at logit 0, then stays in range
    static_assert(PD_MAX_CLUSTER == 8, "a thread per row and CTA");
#pragma unroll
    for (int x = tid; x < 8 * ROWS; x += THREADS) {
        const int r = x >> 3, i = x & 7;
        const bool in = r < rows && i < ctas;
        const float ref1 = in ? ClusterLoad(&ctaRef[r], i) : PD_NO_REF, sum1 = in ? ClusterLoad(&ctaSum[r], i) : 0.0f;
        float m = fmaxf(ref1, -60.0f);
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        }
        const float f = Exp2(ref1 - m);
        float s = f * sum1;
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, o);
        }
        s += Exp2(-m);
        if (r < rows) {
            factorOf[r][i] = f / s;
            if (i == 0) {
                lseOf[r] = m + Log2(s);
            }
        }
    }
    __syncthreads();
    for (int x = rank * THREADS + tid; x < rows * D; x += ctas * THREADS) {
        const int r = x / D, i = x % D;
        const int d = (i >> 1 & 7) * (D / 8) + 2 * (i >> 4) + (i & 1);
        float a = 0;
        if (ctas == 1) {
            a = factorOf[r][0] * accOf[0][r][i];
        } else {
            float accs[PD_MAX_CLUSTER];
#pragma unroll
            for (int j = 0; j < PD_MAX_CLUSTER; ++j) {
                accs[j] = j < ctas ? ClusterLoad(&accOf[0][r][i], j) : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < PD_MAX_CLUSTER; ++j) {
                a = j < ctas ? fmaf(factorOf[r][j], accs[j], a) : a;
            }
        }
        StoreFromFloat(p.Out.Row(seq), (firstHead + r) * D + d, p.OutDtype, a);
    }
    if (track) {
        // one unit per key head: nobody else adds to them
#pragma unroll
        for (int i = 0; i < OWN_KEYS; ++i) {
            const int key = keyFirst + i * THREADS + tid;
            if (slotAt[i] != NOWHERE) {
                float w = 0;
#pragma unroll 4
                for (int r = 0; r < rows; ++r) {
                    w += Exp2(logits[r * p.LogitRow + key - segBeg * PD_TILE] - lseOf[r]);
                }
                c.Weight[slotAt[i]] = before[i] + w;
            }
        }
    }
    if (ctas > 1) {
        ClusterSync(); // no CTA leaves while another reads its shared memory
    }
}

// where a sequence's places begin in the row of all, and how long the ranges are; by one warp
__device__ __forceinline__ void SeqStart(const TPagedDecodeParams &p, int seq, int lane, unsigned ctas, unsigned *start, unsigned *per)
{
    unsigned before = 0, all = 0;
    for (int s = lane; s < p.NSeq; s += 32) {
        const unsigned n = UnitPlaces(SeqTiles<PD_RANGE_TILE>(p, s));
        before += s < seq ? n : 0;
        all += n;
    }
    const int units = p.C.KvHeads * p.HeadChunks;
    *start = __reduce_add_sync(0xffffffffu, before) * units;
    *per = RangePlaces(__reduce_add_sync(0xffffffffu, all) * units, ctas);
}

// records base + i * stride, i = first, first + step, ..: their sums of 4 dimensions (column 4 sub) and of the weights, relative to m
template <int D>
__device__ __forceinline__ void AddRecords(const float *base, size_t stride, int chunks, int first, int step, int sub, float &m, float &l, float4 &acc)
{
    for (int i = first; i < chunks; i += 4 * step) {
        float2 ml[4];
        float4 v[4];
        float top = m;
#pragma unroll
        for (int j = 0; j < 4; ++j) { // four at a time are on their way
            const bool in = i + j * step < chunks;
            const float *src = base + (in ? i + j * step : i) * stride;
            ml[j] = *reinterpret_cast<const float2 *>(src + D);
            v[j] = *reinterpret_cast<const float4 *>(src + 4 * sub);
            ml[j].x = in ? ml[j].x : -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            top = fmaxf(top, ml[j].x);
        }
        const float f = Exp2(m - top);
        m = top;
        l *= f;
        acc = make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (i + j * step < chunks) {
                const float w = Exp2(ml[j].x - m);
                l = fmaf(w, ml[j].y, l);
                acc = make_float4(fmaf(w, v[j].x, acc.x), fmaf(w, v[j].y, acc.y), fmaf(w, v[j].z, acc.z), fmaf(w, v[j].w, acc.w));
            }
        }
    }
}

// Behind the ranges: joins the units that range borders cut, the records in the order of the ranges, and adds the sink.  Few units, many
// records of each (byUnit): a CTA has one row of one unit.  Otherwise CTA b has the unit that border b is the first to cut, a group of
// D / 4 threads a row at a time.  Also writes the zeros of sequences without keys.  A chain of loads, 2.8 us behind the ranges.  The whole call by
// unit and by border, in us: 8 units of 20000 slots 13.1 and 18.3, 64 of 8200 28.8 and 30.1, 128 of 8200 49.6 and 49.2; with eight query heads 14.5 and
// 19.8, 30.2 and 30.4, 53.5 and 51.2.
constexpr int FIN_THREADS = 256;
template <int D>
__global__ void __launch_bounds__(FIN_THREADS) PagedJoinKernel(const TPagedDecodeParams p, unsigned ctas, bool byUnit)
{
    constexpr int LPC = D / 4, GROUPS = FIN_THREADS / LPC;
    __shared__ float refOf[GROUPS], sumOf[GROUPS];
    __shared__ float4 accOf[GROUPS][LPC];
    const int tid = threadIdx.x, lane = tid & 31;
    // the lengths were there before the kernel whose sums are joined began: all that follows from them is worked out before it ends
    TSegment seg = {};
    unsigned start, per;
    int first = 0, chunks = 0; // records of the unit
    if (byUnit) {
        const int units = p.C.KvHeads * p.HeadChunks, unit = blockIdx.x / p.Rows;
        seg.Seq = unit / units;
        seg.Unit = unit % units;
        SeqStart(p, seg.Seq, lane, ctas, &start, &per);
        seg.Keys = SeqTiles<PD_RANGE_TILE>(p, seg.Seq);
        if (seg.Keys.Count > 0) {
            start += (unsigned)seg.Unit * UnitPlaces(seg.Keys) + PD_UNIT_TILES;
            first = start / per;
            chunks = (start + seg.Keys.Count - 1) / per - first + 1;
            chunks = chunks > 1 ? chunks : 0;
        }
    } else if (blockIdx.x > 0) {
        TRangeWalk walk;
        if (walk.Begin(p, lane, blockIdx.x, ctas, false)) {
            seg = walk.Segment(p);
            start = walk.SeqBase + (unsigned)seg.Unit * UnitPlaces(seg.Keys) + PD_UNIT_TILES;
            if (walk.At > start && walk.At - walk.Per <= start) {
                first = blockIdx.x - 1;
                chunks = (start + seg.Keys.Count - 1) / walk.Per - first + 1;
            }
        }
    }
    PdlWait();
    // Not earlier: CTAs of the next call's ranges would come between this kernel's waiting ones, and what those leave on an SM is no room for
    // another range, which then runs alone at the end (512 units of 4000 slots of 64 dimensions: 75 us, 59 this way)
    PdlTrigger();
    for (int s = blockIdx.x; s < p.NSeq; s += gridDim.x) {
        if (SeqTiles<PD_RANGE_TILE>(p, s).Count == 0) {
            for (int x = tid; x < p.HeadCount * D; x += FIN_THREADS) {
                StoreFromFloat(p.Out.Row(s), x, p.OutDtype, 0.0f);
            }
        }
    }
    if (chunks == 0) {
        return;
    }
    const int group = tid / LPC, sub = tid % LPC;
    const int firstHead = seg.Unit / p.HeadChunks * p.Group + seg.Unit % p.HeadChunks * PD_ROWS;
    const int rows = min(p.Group - seg.Unit % p.HeadChunks * PD_ROWS, PD_ROWS);
    const float *base = PartialRecord(p, D, first, seg.Seq, seg.Unit, 0);
    const size_t stride = (size_t)p.Rows * (D + 4);
    if (!byUnit) {
        for (int r = group; r < rows; r += GROUPS) {
            float m = -60.0f, l = 0;
            float4 acc = make_float4(0, 0, 0, 0);
            AddRecords<D>(base + r * (D + 4), stride, chunks, 0, 1, sub, m, l, acc);
            l += Exp2(-m);
            const float v[4] = {acc.x, acc.y, acc.z, acc.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                StoreFromFloat(p.Out.Row(seg.Seq), (firstHead + r) * D + 4 * sub + i, p.OutDtype, v[i] / l);
            }
            if (p.Lse && sub == 0) {
                p.Lse[(size_t)seg.Seq * p.HeadCount + firstHead + r] = m + Log2(l);
            }
        }
        return;
    }
    const int r = blockIdx.x % p.Rows;
    if (r >= rows) {
        return;
    }
    float m = -60.0f, l = 0;
    float4 acc = make_float4(0, 0, 0, 0);
    AddRecords<D>(base + r * (D + 4), stride, chunks, group, GROUPS, sub, m, l, acc);
    accOf[group][sub] = acc;
    if (sub == 0) {
        refOf[group] = m;
        sumOf[group] = l;
    }
    __syncthreads();
    if (tid < D) {
        m = refOf[0];
#pragma unroll
        for (int i = 1; i < GROUPS; ++i) {
            m = fmaxf(m, refOf[i]);
        }
        l = Exp2(-m);
        float a = 0;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            const float f = Exp2(refOf[i] - m);
            l = fmaf(f, sumOf[i], l);
            a = fmaf(f, reinterpret_cast<const float *>(accOf[i])[tid], a);
        }
        StoreFromFloat(p.Out.Row(seg.Seq), (firstHead + r) * D + tid, p.OutDtype, a / l);
        if (p.Lse && tid == 0) {
            p.Lse[(size_t)seg.Seq * p.HeadCount + firstHead + r] = m + Log2(l);
        }
    }
}

// weight += sum over the query heads of a key head of 2^(z - log2 of all weights and the sink): four slots per thread.  What does not come
// from the kernels before (the lengths, the table, the weights, which only this kernel writes) is loaded before they end.  It reads and writes
// 8 bytes a slot and 4 a logit: 7 us behind the join for 40 x 8 key heads of 2048 .. 6144 slots, four query heads each (inside the join instead: 15 to 18).
constexpr int WGT_THREADS = 256, WGT_SLOTS = 4 * WGT_THREADS;
__global__ void __launch_bounds__(WGT_THREADS) PagedWeightKernel(const TPagedDecodeParams p)
{
    const TPages &c = p.C;
    const int kvHead = blockIdx.y, seq = blockIdx.z, slot = blockIdx.x * WGT_SLOTS + 4 * threadIdx.x;
    const TSeqKeys keys = SeqTiles<PD_RANGE_TILE>(p, seq);
    const int first = keys.First * PD_RANGE_TILE; // slots that the ranges did not look at have no logits
    const int page = slot < keys.End && slot + 3 >= first ? c.Table.Row(seq)[slot >> c.PageShift] : -1;
    const bool in = (unsigned)page < (unsigned)c.PageCount;
    float *const dst = c.Weight + PlaneSlot(c, in ? page : 0, kvHead) + (slot & ((1 << c.PageShift) - 1));
    float4 w = make_float4(0, 0, 0, 0);
    if (in) {
        w = *reinterpret_cast<const float4 *>(dst);
    }
    PdlWait();
    PdlTrigger();
    if (!in) {
        return;
    }
    const size_t head = (size_t)seq * p.HeadCount + kvHead * p.Group;
    const float *lse = p.Lse + head, *z = p.Logits + head * p.LogitRow + slot;
    const bool whole = slot >= first && slot + 3 < keys.End;
#pragma unroll 4
    for (int r = 0; r < p.Group; ++r) {
        float4 x = *reinterpret_cast<const float4 *>(z + (size_t)r * p.LogitRow);
        const float l = lse[r];
        if (!whole) {
            x.x = slot >= first && slot < keys.End ? x.x : -INFINITY;
            x.y = slot + 1 >= first && slot + 1 < keys.End ? x.y : -INFINITY;
            x.z = slot + 2 >= first && slot + 2 < keys.End ? x.z : -INFINITY;
            x.w = slot + 3 >= first && slot + 3 < keys.End ? x.w : -INFINITY;
        }
        w.x += Exp2(x.x - l);
        w.y += Exp2(x.y - l);
        w.z += Exp2(x.z - l);
        w.w += Exp2(x.w - l);
    }
    *reinterpret_cast<float4 *>(dst) = w;
}

// Which form a call takes.  Clusters of CTAs of two to eight tiles per warp while all of them are resident (four to an SM, three where more than
// eight heads share a key head; of eight CTAs, which have to lie in one part of the chip, on 128 of the SMs), with fewer CTAs of a unit where that
// makes them so.  Measured, in us, as clusters and as ranges, for units of two int8 heads of 128 dimensions (8 key heads a sequence):
//   units x slots      8 x 256    64 x 1024   64 x 4000   72 x 1024 (of 4)  128 x 512   256 x 256   256 x 1024 (of 2: left to the ranges)
//   clusters / ranges  5.5 / 6.6  7.4 / 9.1   14.9 / 15.4     9.0 / 9.7     7.6 / 9.7   7.4 / 8.8   26.9 / 15.8
// Beyond the resident ones a CTA per unit pays while it has few tiles, 24 of 128 dimensions or 32 of 64:
//   heads of a unit x D   2 x 128                                    16 x 128                        16 x 64, with weights        4 x 64
//   units x slots         1024 x 256  1024 x 512  2048 x 512         664 x 384  2048 x 384           664 x 512  2048 x 512        664 x 512  2048 x 512
//   clusters / ranges     17.0 / 20.9  31.0 / 32.0  58 / 54          27.7 / 32.3  74 / 68            23.4 / 41.5  65 / 103        15.6 / 19.6  40 / 44
// Units that share a key head's weights leave them to the kernel behind the ranges.
struct TPagedForm {
    int Cluster; // CTAs of a unit; 0: ranges
    // parts of the workspace, in this order
    size_t Partial, Lse, Logits, Bytes;
    int LogitRow;
    int ListCap; // keys that a CTA lists; 0: none
    bool OneWarp; // of a CTA
};
constexpr int PD_SPARSE_MIN = 1024, PD_SPARSE_SLOTS = 512;
constexpr int B200_SMS = 148, PD_MAX_CLUSTER_SMS = 128;
static TPagedForm PagedForm(int headDim, int nSeq, int kvHeads, int headCount, int maxCtx, int window, bool positions, bool track)
{
    auto round = [](size_t x) { return (x + 255) / 256 * 256; };
    const int group = headCount / kvHeads, rows = group < PD_ROWS ? group : PD_ROWS, chunks = (group + PD_ROWS - 1) / PD_ROWS;
    const size_t units = (size_t)nSeq * kvHeads * chunks;
    // keys of a sequence that a call looks at
    const long long keysMax = positions ? maxCtx : window == 0 ? 1 : maxCtx < window ? maxCtx : window;
    const long long tilesMax = (keysMax + PD_TILE - 1) / PD_TILE + 1;
    TPagedForm w;
    w.Cluster = 1;
    while (w.Cluster < PD_MAX_CLUSTER && tilesMax > (PD_MIN_TILES + 1) * w.Cluster) {
        w.Cluster *= 2;
    }
    auto resident = [&] { return units * w.Cluster <= (size_t)(w.Cluster == PD_MAX_CLUSTER ? PD_MAX_CLUSTER_SMS : B200_SMS) * (rows > 8 ? 3 : 4); };
    while (w.Cluster > 1 && !resident()) {
        w.Cluster /= 2;
    }
    const bool inTime = resident() && tilesMax <= 4 * PD_MIN_TILES * w.Cluster, one = w.Cluster == 1 && tilesMax <= (headDim == 64 ? 4 : 3) * PD_MIN_TILES + 1;
    if (!(inTime || one) || (track && chunks > 1)) {
        w.Cluster = 0;
    }
    // A window much shorter than a cache with positions: its keys may be anywhere, so all slots have to be looked at, but only by their positions, and
    // the window's rows alone are read.  Pays from half the cache on against the ranges, a quarter against clusters that read all, which are short of
    // bytes to save and have no list to wait for.  Measured with and without, in us, units of four int8 heads x 128, windows 64 / 1000:
    //   units x slots   4 x 8192         32 x 4096         128 x 8192        512 x 3000         1024 x 8192      32 x 400000
    //   with            7.2 / 9.5        7.9 / 10.9        9.7 / 17.0        12.4 / 36.7        34 / 92          47 / 60
    //   without         11.5 / 11.6      14.0 / 14.0       42.8 / 42.6       62.6 / 62.5        278 / 278        401 / 401
    // 512 slots to a CTA (1024: 4 units of 1500 slots, window 250, 9.2 instead of 8.1), as far as eight CTAs go.  (resident() counts four or three CTAs
    // to an SM here too, where list and logits may leave place for fewer: sixteen heads x 128 with weights, window 1000, take 112 KB, so that 296 units of 4096
    // slots take 42 us and 304 76.)
    w.ListCap = 0;
    const int listMax = window == 0 ? 1 : window;
    if (positions && listMax <= PD_MAX_LIST && maxCtx > PD_SPARSE_MIN && maxCtx / listMax >= (w.Cluster ? 4 : 2) && !(track && chunks > 1)) {
        w.Cluster = 1;
        while (w.Cluster < PD_MAX_CLUSTER && maxCtx > PD_SPARSE_SLOTS * w.Cluster) {
            w.Cluster *= 2;
        }
        while (w.Cluster > 1 && !resident()) {
            w.Cluster /= 2;
        }
        w.ListCap = (listMax + PD_TILE - 1) / PD_TILE * PD_TILE;
    }
    // A warp per unit where CTAs of four would come in more than one and a half turns, or in more than one for a tile or two of narrow units.
    // Measured, in us, with one warp and with four, 128 int8 dimensions, two / sixteen query heads a unit: 640 units of 16 slots 5.8, 7.7 / 16.3, 14.9; 1024 of 64
    // 9.4, 10.0 / 20.6, 23.2; 2048 of 16 7.1, 15.4 / 31, 36; 2048 of 112 14.5, 21.7 / 44.5, 46.2
    const size_t four = (size_t)B200_SMS * (rows > 8 ? 3 : 4);
    w.OneWarp = w.Cluster == 1 && w.ListCap == 0 && tilesMax <= PD_ONE_WARP_TILES && (2 * units > 3 * four || (units > four && rows <= 8 && tilesMax <= 3));
    // clusters: of a CTA, an odd number of tiles, so that the rows of a store lie in different banks
    w.LogitRow = w.ListCap ? (w.ListCap / PD_TILE | 1) * PD_TILE : w.Cluster ? (int)((tilesMax + w.Cluster - 1) / w.Cluster | 1) * PD_TILE
                           : (int)((maxCtx < 0x7ffffff0 ? (long long)maxCtx + PD_TILE - 1 : 0x7ffffff0ll) / PD_TILE * PD_TILE);
    w.Partial = 0;
    w.Lse = w.Logits = w.Bytes = 0; // a cluster has all it needs in shared memory
    if (!w.Cluster) {
        w.Lse = round((PD_MAX_CTAS + units) * rows * (headDim + 4) * sizeof(float));
        w.Logits = w.Lse + (track ? round((size_t)nSeq * headCount * sizeof(float)) : 0);
        w.Bytes = w.Logits + (track ? (size_t)nSeq * headCount * w.LogitRow * sizeof(float) : 0);
    }
    return w;
}

template <int D, bool E4M3, bool SPARSE, int WARPS>
static const void *PickWidth(bool f16, bool wide)
{
    return f16 ? (wide ? (const void *)PagedClusterKernel<D, E4M3, true, true, SPARSE, WARPS> : (const void *)PagedClusterKernel<D, E4M3, true, false, SPARSE, WARPS>)
               : (wide ? (const void *)PagedClusterKernel<D, E4M3, false, true, SPARSE, WARPS> : (const void *)PagedClusterKernel<D, E4M3, false, false, SPARSE, WARPS>);
}
template <int D, bool E4M3>
static const void *PickCluster(bool f16, bool wide, bool sparse, bool oneWarp)
{
    return sparse ? PickWidth<D, E4M3, true, PD_WARPS>(f16, wide) : oneWarp ? PickWidth<D, E4M3, false, 1>(f16, wide) : PickWidth<D, E4M3, false, PD_WARPS>(f16, wide);
}

} // namespace tsa

using namespace tsa;

extern "C" __attribute__((visibility("default"))) size_t tsa_paged_decode_workspace_bytes(const tsa_paged_cfg *cfg, const tsa_paged_kv *kv, int nSeq, int headCount,
    int maxCtx, int window)
{
    if (!cfg || !kv || nSeq <= 0 || kv->kv_heads <= 0 || headCount < kv->kv_heads || maxCtx < 0 || window < 0) {
        return 0;
    }
    return PagedForm(cfg->head_dim, nSeq, kv->kv_heads, headCount, maxCtx, window, kv->pos != nullptr, kv->weight != nullptr).Bytes;
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
    const bool track = kv->weight != nullptr;
    const long long room = TableTokens(p.C);
    const int longest = room < maxCtx ? (int)room : maxCtx;
    const long long units = (long long)nSeq * kv->kv_heads * p.HeadChunks, tilesMax = (long long)longest / PD_TILE + 8;
    TSA_REQUIRE(units * tilesMax < (1ll << 31), "tsa_paged_decode: %d sequences of %d tokens with %d query heads are too much for one call", nSeq, longest, headCount);
    const TPagedForm form = PagedForm(D, nSeq, kv->kv_heads, headCount, maxCtx, window, kv->pos != nullptr, track);
    TSA_REQUIRE(form.Bytes == 0 || (workspace && workspaceBytes >= form.Bytes), "tsa_paged_decode: workspace of %zu bytes needed, %zu given", form.Bytes, workspaceBytes);
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
    p.Lse = track ? (float *)((char *)workspace + form.Lse) : nullptr;
    p.Logits = track ? (float *)((char *)workspace + form.Logits) : nullptr;
    p.LogitRow = form.LogitRow;
    p.ListCap = form.ListCap;
    p.Status = statusWord;
    p.Cluster = form.Cluster;
    const bool e4m3 = cfg->kv_dtype == TSA_E4M3, f16 = cfg->scale_dtype == TSA_F16;
    p.ScaleF16 = f16;
    cudaStream_t s = (cudaStream_t)stream;
    if (form.Cluster) {
        const bool wide = p.Group > 8;
        const bool sparse = form.ListCap > 0;
        const void *kern = D == 128 ? (e4m3 ? PickCluster<128, true>(f16, wide, sparse, form.OneWarp) : PickCluster<128, false>(f16, wide, sparse, form.OneWarp))
                                    : (e4m3 ? PickCluster<64, true>(f16, wide, sparse, form.OneWarp) : PickCluster<64, false>(f16, wide, sparse, form.OneWarp));
        const size_t smem = (track ? p.Rows * form.LogitRow * sizeof(float) : 0) + form.ListCap * (sizeof(size_t) + sizeof(int));
        if (smem > 0 && (wide || sparse)) { // beyond 48 KB with what the kernel has anyway; the same limit in every call
            const int most = sparse ? PD_MAX_LIST : 4 * PD_MIN_TILES * PD_TILE;
            rc = CheckCuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                (wide ? PD_ROWS : 8) * (most + PD_TILE) * (int)sizeof(float) + (sparse ? PD_MAX_LIST * (int)(sizeof(size_t) + sizeof(int)) : 0)), "cudaFuncSetAttribute");
            if (rc != TSA_OK) {
                return rc;
            }
        }
        void *args[] = {&p};
        return CheckCuda(LaunchPdl(kern, dim3((unsigned)(units * p.Cluster)), dim3(form.OneWarp ? 32 : PD_WARPS * 32), smem, s, args, p.Cluster), "tsa_paged_decode launch");
    }
    unsigned ctas = 0;
    rc = LaunchPagedRanges(p, kv, D, e4m3, (long long)(p.C.Pos || longest < window ? longest : window) / PD_RANGE_TILE + 2, &ctas, s);
    if (rc == TSA_OK) {
        const void *join = D == 128 ? (const void *)PagedJoinKernel<128> : (const void *)PagedJoinKernel<64>;
        bool byUnit = units * 4 < ctas;
        void *args[] = {&p, &ctas, &byUnit};
        rc = CheckCuda(LaunchPdl(join, dim3(byUnit ? (unsigned)units * p.Rows : ctas), dim3(FIN_THREADS), 0, s, args), "tsa_paged_decode join launch");
    }
    if (rc == TSA_OK && track && longest > 0) {
        void *args[] = {&p};
        rc = CheckCuda(LaunchPdl((const void *)PagedWeightKernel, dim3((longest + WGT_SLOTS - 1) / WGT_SLOTS, kv->kv_heads, nSeq), dim3(WGT_THREADS), 0, s, args),
            "tsa_paged_decode weights launch");
    }
    return rc;
}

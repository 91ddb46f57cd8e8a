// Attention of one new token per sequence over the paged cache, on the 5th-generation tensor cores: the form for long caches and large
// batches (paged_decode.cu has the mathematics and the form for short ones).
//
// What bounds it is the stream of the cache, so nothing but the copy engine and the tensor cores touches the codes of K and V:
//   scores  [128 keys][16 heads]      = K tile [128][D] (shared memory, as the pages hold it) * q [16][D]
//   result  [D][16 columns per 4 heads] += V tile [128][D] read along its rows * weights [128 keys][16 columns per 4 heads]
// kind::i8 or kind::f8f6f4, accumulators in tensor memory.  A weight w = 2^(z - ref) * vScale, |w| < 2^4, is four columns of 8 bits that
// add up to it: for int8 the signed base-256 digits of w * 2^27 (off by 2^-28), for e4m3 the roundings of w * 2^4 and of what the digits
// before left over, 32 times larger each (off by 2^-16 of w, or by 2^-29 if that is more).  The columns cost the tensor cores nothing that
// shows: 128 x D x 64 per 33 KB of cache.  Each of the 128 arithmetic threads has one key of the tile and the weights of all heads for it.
//
// Measured: 64 sequences of 1024 .. 8192 slots, 16 key heads x 128 int8, 1.31 GB: 181 to 205 us, 6.4 to 7.2 TB/s (a plain copy: 6.45; mma.sync with
// the codes in registers: 213 us); 48 of 500 .. 9000, 8 key heads x 128 e4m3 of four query heads, 0.5 GB: 84 to 94; 2 of 100000 .. 131072, 4 key heads of eight
// query heads, 0.27 GB: 48.  What short calls lose is the start (lengths, page, first tile: 4 us) and the join; the tensor pipe is at 4 to 6 %, the
// issue slots at 23 (128 dimensions, up to four heads a unit) to 41 % (64).
//
// One CTA: a warp that issues the copies (a box per page, up to 128 slots; tiles ahead of the arithmetic as far as the ring goes, across
// units), one that issues the products, four for the weights.  Two CTAs per SM: while one of them ends a unit, the other has the memory.
// Three where a tile is half as large and the weights leave the room (64 dimensions, up to eight heads): 512 key heads of 4000 slots 54 us instead of 61.
// What the digits leave out is absolute, so that very many light keys behind a heavy one would be lost beside a reference that only rises (131072
// keys of 2^-22 of the first: 0.6 % of the sum with int8, 2.5 % with e4m3).  The sums therefore leave tensor memory for registers, which hold them in
// float32, every 16 tiles, and when a weight would exceed 2^4; the accumulation then starts anew with the largest weight of the present tile as the
// reference, be it higher or lower.  2048 keys are off by 2^-17 of 2^ref at most, a key among them weighs half of that or more: 2^-16 of the sum of the
// weights, however many the keys.  References are whole numbers, so that the sums are scaled without roundings.  All waits are bounded.
#include "att_sm100_common.cuh"
#include "paged_decode.cuh"

namespace tsa {

constexpr int PT_SOFT_WARPS = 4, PT_LOAD_WARP = 4, PT_MMA_WARP = 5;
constexpr int PT_THREADS = 6 * 32;
constexpr int PT_SOFT_THREADS = PT_SOFT_WARPS * 32;
constexpr int PT_KEYS = PD_RANGE_TILE;
constexpr int PT_TMEM_COLS = 128;         // scores twice 16, result up to 64
constexpr int PT_DRAIN_TILES = 16;        // int32 would overflow after 1024 (digits * codes up to 2^14)
constexpr float PT_EDGE = 4.0f - 1.0f / 64; // log2 of the largest weight: the digits of int8 end at 2^4 * 0.996
constexpr float PT_I8_UNIT = 1 << 27, PT_E4M3_UNIT = 16.0f; // what a weight of 1 is in digits
constexpr float PT_E4M3_STEP = 32.0f;     // from a digit to the next: roundings of numbers up to 256 leave 8 at most, so that the next is up to 256 again
// log2 of what a reference may lie below the range's highest: 2^30 keys of 2^(84 + 12) each can still be summed in float32, and of keys far below that
// one 8 million are off by 2^-17 of it
constexpr float PT_SINK = 12.0f;

// what the weights need of a tile's keys besides their scores
struct TTileKeys {
    float KScale[PT_KEYS], VScale[PT_KEYS];
    float Bias[PT_KEYS]; // slope * distance; infinity: the key is masked
};

template <int D, int HB>
struct TTcLayout {
    static constexpr int TILE_BYTES = PT_KEYS * D;
    static constexpr int CTAS = D == 64 && HB < 4 ? 3 : 2; // per SM
    static constexpr int STAGES = D == 64 && HB == 4 ? 5 : 3; // of the ring of K and V tiles
    static constexpr int RING_BYTES = STAGES * 2 * TILE_BYTES;
    static constexpr int Q_BYTES = PD_ROWS * D;
    static constexpr int W_BYTES = HB * PT_KEYS * 16;
    static constexpr int W_BUFS = D == 128 && HB == 4 ? 1 : 2; // as many as leave two CTAs their shared memory
    static constexpr int KEY_BYTES = STAGES * (int)sizeof(TTileKeys);
    static constexpr int BYTES = RING_BYTES + Q_BYTES + W_BUFS * W_BYTES + KEY_BYTES + 1024; // the base is rounded up to 1024
};

template <int STAGES>
struct TTcMisc {
    uint64_t Full[STAGES], Empty[STAGES], KeysFull[STAGES];
    uint64_t SReady[2], SFree[2], WReady[2], WFree[2], QReady, Done;
    uint32_t TmemBase;
    int Abort;
    int Fresh[2];                // the product with these weights starts a new sum
    alignas(16) float Mult[2][PD_ROWS];     // query scale times the logits' factor, of this unit and the next
    alignas(16) float Ref[PD_ROWS];
    float Top[PD_ROWS];          // the highest reference so far
    float Red[PT_SOFT_WARPS][PD_ROWS];
    alignas(16) float Factor[PD_ROWS];
};

// or over the arithmetic threads; a barrier among them
__device__ __forceinline__ bool SoftAny(bool x)
{
    int r;
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        "setp.ne.b32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, 1, %2, p;\n\t"
        "selp.b32 %0, 1, 0, q;\n\t"
        "}"
        : "=r"(r)
        : "r"((int)x), "n"(PT_SOFT_THREADS)
        : "memory");
    return r != 0;
}

// two weights' next e4m3 digits; a and b become PT_E4M3_STEP times what is left over
__device__ __forceinline__ uint32_t TakeDigit(float &a, float &b)
{
    const uint32_t d = PackE4M3x2(a, b);
    const float2 f = UnpackE4M3x2(d);
    a = (a - f.x) * PT_E4M3_STEP;
    b = (b - f.y) * PT_E4M3_STEP;
    return d;
}

// 2^n of a whole number up to 127, without a rounding; 0 below 2^-126
__device__ __forceinline__ float WholeExp2(float n)
{
    return n < -126.0f ? 0.0f : __int_as_float(((int)n + 127) << 23);
}

// floats as integers of the same order
__device__ __forceinline__ int OrderedInt(float x)
{
    const int b = __float_as_int(x);
    return b ^ (b >> 31 & 0x7fffffff);
}
__device__ __forceinline__ float FromOrderedInt(int b)
{
    return __int_as_float(b ^ (b >> 31 & 0x7fffffff));
}

// sums over the warp of N values per lane (N a power of two): lanes keep half of the values at each step, so that N + 4 shuffles do for
// N = 16 where one sum after the other takes 5 N.  The sum of value HeadOfLane<N>(lane) ends up in v[0].
template <int N>
__device__ __forceinline__ int HeadOfLane(int lane)
{
    return N == 16 ? lane >> 1 : N == 8 ? lane >> 2 : lane >> 3;
}
template <int N>
__device__ __forceinline__ void WarpSums(float (&v)[N], int lane)
{
    int mask = 16;
#pragma unroll
    for (int n = N / 2; n >= 1; n /= 2, mask /= 2) {
        const bool upper = lane & mask;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const float send = upper ? v[i] : v[i + n], keep = upper ? v[i + n] : v[i];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, send, mask);
        }
    }
#pragma unroll
    for (; mask >= 1; mask /= 2) {
        v[0] += __shfl_xor_sync(0xffffffffu, v[0], mask);
    }
}

// HB: blocks of four query heads (1, 2 or 4)
template <int D, bool E4M3, int HB>
__global__ void __launch_bounds__(PT_THREADS, (TTcLayout<D, HB>::CTAS)) PagedRangeKernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
    const TPagedDecodeParams p)
{
    typedef TTcLayout<D, HB> TL;
    constexpr int STAGES = TL::STAGES, W_BUFS = TL::W_BUFS, HEADS = 4 * HB;
    constexpr uint32_t IDESC_QK = E4M3 ? MakeInstrDesc(1, 0, 0, 0, 0, PT_KEYS, PD_ROWS) : MakeInstrDesc(2, 1, 1, 0, 0, PT_KEYS, PD_ROWS);
    constexpr uint32_t IDESC_WV = E4M3 ? MakeInstrDesc(1, 0, 0, 1, 1, D, 16 * HB) : MakeInstrDesc(2, 1, 1, 1, 1, D, 16 * HB);
    extern __shared__ uint8_t rawShared[];
    __shared__ TTcMisc<STAGES> misc;
    uint8_t *const smem = rawShared + ((1024 - (SmemAddr(rawShared) & 1023)) & 1023);
    uint8_t *const qTile = smem + TL::RING_BYTES, *const wTile = qTile + TL::Q_BYTES;
    TTileKeys *const tileKeys = reinterpret_cast<TTileKeys *>(wTile + W_BUFS * TL::W_BYTES);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const TPages &c = p.C;

    if (tid == 0) {
        for (int i = 0; i < STAGES; ++i) {
            MbarInit(&misc.Full[i], 1);
            MbarInit(&misc.Empty[i], 1);
            MbarInit(&misc.KeysFull[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            MbarInit(&misc.SReady[i], 1);
            MbarInit(&misc.SFree[i], PT_SOFT_THREADS);
            MbarInit(&misc.WReady[i], PT_SOFT_THREADS);
            MbarInit(&misc.WFree[i], 1);
        }
        MbarInit(&misc.QReady, PT_SOFT_THREADS);
        MbarInit(&misc.Done, 1);
        misc.Abort = 0;
        FenceBarrierInit();
    }
    if (warp == PT_MMA_WARP) {
        TmemAlloc(&misc.TmemBase, PT_TMEM_COLS);
        TmemRelinquish();
    }
    if (warp == PT_LOAD_WARP && lane == 0) {
        PrefetchTensorMap(&tmK);
        PrefetchTensorMap(&tmV);
    }
    TcFenceBefore();
    __syncthreads();
    TcFenceAfter();
    const uint32_t tmem = misc.TmemBase, tmemOut = tmem + 32;
    const int *abortFlag = &misc.Abort;
    auto fail = [&](int code) {
        *(volatile int *)&misc.Abort = 1;
        if (p.Status) {
            atomicOr(p.Status, code);
        }
    };
    PdlWait();
    PdlTrigger(); // behind the allocation of tensor memory

    TRangeWalk walk;
    const bool any = walk.Begin(p, lane, blockIdx.x, gridDim.x, blockIdx.x == 0 && warp == 0);
    if (!any) {
        // nothing: on to the end
    } else if (warp == PT_LOAD_WARP) {
        // ---- copies; scales and masks of the keys, four to a lane
        const int boxShift = min(c.PageShift, 7), boxes = PT_KEYS >> boxShift;
        const int noRow = (int)(((long long)c.PageCount * c.KvHeads) << c.PageShift); // a box from here on is zeros
        const int nearest = p.Window > 0 ? 1 : 0;
        const unsigned spread = p.Window > 0 ? p.Window : 1;
        int count = 0;
        bool ok = true, badPage = false;
        uint4 rawK = make_uint4(0, 0, 0, 0), rawV = make_uint4(0, 0, 0, 0); // scales of the tile before, on their way
        int4 pos = make_int4(0, 0, 0, 0);
        bool pageOk = false;
        TSegment seg = walk.Segment(p);
        int head = 0, cur = 0;
        const int *table = nullptr;
        auto pageOf = [&](int tile) {
            const int slot = tile * PT_KEYS + 4 * lane;
            return tile < seg.TileEnd && slot < seg.Keys.End ? table[slot >> c.PageShift] : -1;
        };
        auto load = [&](int tile, int page) {
            pageOk = (unsigned)page < (unsigned)c.PageCount;
            const int slot = tile * PT_KEYS + 4 * lane;
            if (pageOk) {
                const size_t at = PlaneSlot(c, page, head) + (slot & ((1 << c.PageShift) - 1));
                if (p.ScaleF16) {
                    const uint2 k = *reinterpret_cast<const uint2 *>(c.KScale + at * 2), v = *reinterpret_cast<const uint2 *>(c.VScale + at * 2);
                    rawK.x = k.x;
                    rawK.y = k.y;
                    rawV.x = v.x;
                    rawV.y = v.y;
                } else {
                    rawK = *reinterpret_cast<const uint4 *>(c.KScale + at * 4);
                    rawV = *reinterpret_cast<const uint4 *>(c.VScale + at * 4);
                }
                if (c.Pos) {
                    pos = *reinterpret_cast<const int4 *>(c.Pos + at);
                }
            } else {
                badPage |= slot < seg.Keys.End && slot + 3 >= seg.Keys.Beg;
            }
        };
        auto store = [&](int tile, int n) {
            TTileKeys &keys = tileKeys[n % STAGES];
            const int slot = tile * PT_KEYS + 4 * lane;
            const int at[4] = {c.Pos ? pos.x : slot, c.Pos ? pos.y : slot + 1, c.Pos ? pos.z : slot + 2, c.Pos ? pos.w : slot + 3};
            const uint32_t k[4] = {rawK.x, rawK.y, rawK.z, rawK.w}, v[4] = {rawV.x, rawV.y, rawV.z, rawV.w};
            float ks[4], vs[4], bias[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int far = cur - at[i];
                const bool valid = pageOk && slot + i >= seg.Keys.Beg && slot + i < seg.Keys.End && (unsigned)(far - nearest) < spread;
                ks[i] = p.ScaleF16 ? __half2float(__ushort_as_half((unsigned short)(i & 1 ? k[i / 2] >> 16 : k[i / 2] & 0xffff))) : __uint_as_float(k[i]);
                vs[i] = p.ScaleF16 ? __half2float(__ushort_as_half((unsigned short)(i & 1 ? v[i / 2] >> 16 : v[i / 2] & 0xffff))) : __uint_as_float(v[i]);
                vs[i] = valid ? vs[i] : 0.0f;
                // + 0 * vs: a value scale that is no number makes the weights none, which the sum of weights then shows
                bias[i] = valid ? fmaf(p.Slope, (float)far, vs[i] * 0.0f) : INFINITY;
            }
            *reinterpret_cast<float4 *>(&keys.KScale[4 * lane]) = make_float4(ks[0], ks[1], ks[2], ks[3]);
            *reinterpret_cast<float4 *>(&keys.VScale[4 * lane]) = make_float4(vs[0], vs[1], vs[2], vs[3]);
            *reinterpret_cast<float4 *>(&keys.Bias[4 * lane]) = make_float4(bias[0], bias[1], bias[2], bias[3]);
            __syncwarp();
            if (lane == 0) {
                MbarArrive(&misc.KeysFull[n % STAGES]);
            }
        };
        for (bool more = true; more && ok;) {
            seg = walk.Segment(p);
            head = seg.Unit / p.HeadChunks;
            cur = (p.Tokens ? p.Tokens[seg.Seq] : p.CtxLens[seg.Seq]) - 1;
            table = c.Table.Row(seg.Seq);
            int page = pageOf(seg.TileBeg);
            for (int tile = seg.TileBeg; tile < seg.TileEnd && ok; ++tile, ++count) {
                const int stage = count % STAGES;
                if (tile > seg.TileBeg) {
                    store(tile - 1, count - 1); // under way since the last turn; its place became free then
                }
                load(tile, page);
                // where the boxes are; boxes without keys are zeros
                const int boxPage = __shfl_sync(0xffffffffu, page, (lane << boxShift) / 4 & 31);
                page = pageOf(tile + 1);
                const int slot = tile * PT_KEYS + (lane << boxShift);
                int row = noRow;
                if (lane < boxes && slot + (1 << boxShift) > seg.Keys.Beg && (unsigned)boxPage < (unsigned)c.PageCount) {
                    row = (int)PlaneSlot(c, boxPage, head) + (slot & ((1 << c.PageShift) - 1));
                }
                if (count >= STAGES) {
                    ok = __all_sync(0xffffffffu, WaitBarA(&misc.Empty[stage], (count / STAGES - 1) & 1, abortFlag));
                    if (!ok) {
                        if (lane == 0) {
                            fail(kDevTimeoutMma);
                        }
                        break;
                    }
                }
                uint8_t *k = smem + stage * 2 * TL::TILE_BYTES, *v = k + TL::TILE_BYTES;
                if (lane == 0) {
                    MbarExpectTx(&misc.Full[stage], 2 * TL::TILE_BYTES);
                }
                __syncwarp();
                if (lane < boxes) {
                    TmaLoad2D(k + (lane << boxShift) * D, &tmK, 0, row, &misc.Full[stage]);
                    TmaLoad2D(v + (lane << boxShift) * D, &tmV, 0, row, &misc.Full[stage]);
                }
            }
            if (ok) {
                store(seg.TileEnd - 1, count - 1);
            }
            more = walk.Next(p, seg);
        }
        if (badPage && p.Status) {
            atomicOr(p.Status, kDevBadSpan);
        }
        // no copy is under way when the CTA leaves
        for (int i = max(0, count - STAGES); i < count; ++i) {
            if (!WaitBar(&misc.Full[i % STAGES], (i / STAGES) & 1)) {
                fail(kDevTimeoutTma);
            }
        }
    } else if (warp == PT_MMA_WARP) {
        // ---- products
        constexpr int SWZ = D;
        const uint64_t qDesc = MakeSmemDesc(SmemAddr(qTile), 16, 8 * D, SWZ);
        // weights: 16 columns side by side (16 bytes), 8 keys 128 bytes apart, the next 16 columns behind all keys; no swizzle
        const uint64_t wDesc = MakeSmemDesc(SmemAddr(wTile), 128, PT_KEYS * 16, SWZ) & ~(7ull << 61);
        int count = 0, segments = 0;
        bool ok = true;
        auto wait = [&](uint64_t *bar, uint32_t parity, int code) {
            const bool done = __all_sync(0xffffffffu, WaitBarA<true>(bar, parity, abortFlag));
            if (!done && ok && lane == 0) {
                fail(code);
            }
            ok = ok && done;
            return done;
        };
        // result += V^T * weights of tile number n
        auto weigh = [&](int n) {
            const int buf = n % W_BUFS;
            if (!wait(&misc.WReady[buf], (n / W_BUFS) & 1, kDevTimeoutMma)) {
                return;
            }
            TcFenceAfter();
            const int stage = n % STAGES;
            const uint64_t vDesc = MakeSmemDesc(SmemAddr(smem + stage * 2 * TL::TILE_BYTES + TL::TILE_BYTES), 16, 8 * D, SWZ);
            const uint32_t first = *(volatile int *)&misc.Fresh[buf] ? 0 : 1;
            if (ElectOne()) {
#pragma unroll
                for (int s = 0; s < PT_KEYS / 32; ++s) {
                    const uint64_t a = vDesc + s * (32 * D / 16), b = wDesc + buf * (TL::W_BYTES / 16) + s * (32 * 16 / 16);
                    if (E4M3) {
                        MmaF8SS(tmemOut, a, b, IDESC_WV, s ? 1 : first);
                    } else {
                        MmaI8SS(tmemOut, a, b, IDESC_WV, s ? 1 : first);
                    }
                }
                MmaCommit(&misc.Empty[stage]);
                MmaCommit(&misc.WFree[buf]);
            }
            __syncwarp();
        };
        for (bool more = true; more && ok; ++segments) {
            const TSegment seg = walk.Segment(p);
            for (int tile = seg.TileBeg; tile < seg.TileEnd && ok; ++tile, ++count) {
                const bool newUnit = tile == seg.TileBeg;
                if (newUnit) { // there before the last weights of the unit before
                    wait(&misc.QReady, segments & 1, kDevTimeoutMma);
                }
                const int stage = count % STAGES, buf = count & 1;
                if (!ok || !wait(&misc.Full[stage], (count / STAGES) & 1, kDevTimeoutTma)) {
                    break;
                }
                if (count >= 2 && !wait(&misc.SFree[buf], (count / 2 - 1) & 1, kDevTimeoutMma)) {
                    break;
                }
                TcFenceAfter();
                const uint64_t kDesc = MakeSmemDesc(SmemAddr(smem + stage * 2 * TL::TILE_BYTES), 16, 8 * D, SWZ);
                if (ElectOne()) {
#pragma unroll
                    for (int s = 0; s < D / 32; ++s) {
                        if (E4M3) {
                            MmaF8SS(tmem + buf * 16, kDesc + 2 * s, qDesc + 2 * s, IDESC_QK, s > 0);
                        } else {
                            MmaI8SS(tmem + buf * 16, kDesc + 2 * s, qDesc + 2 * s, IDESC_QK, s > 0);
                        }
                    }
                    MmaCommit(&misc.SReady[buf]);
                }
                __syncwarp();
                if (count > 0) {
                    weigh(count - 1);
                }
            }
            more = walk.Next(p, seg);
        }
        if (ok) {
            weigh(count - 1);
        }
        // nothing is under way when tensor memory is given back
        if (ElectOne()) {
            MmaCommit(&misc.Done);
        }
        __syncwarp();
        if (!WaitBar(&misc.Done, 0)) {
            fail(kDevTimeoutMma);
        }
    } else {
        // ---- weights: one key per thread
        const uint32_t laneBase = (uint32_t)(warp * 32) << 16;
        // dimension of this thread's lane of the result: all 128 lanes, or 16 of each warp's
        const int dim = D == 128 ? tid : warp * 16 + lane;
        const bool hasDim = D == 128 || lane < 16;
        int count = 0, segments = 0;
        bool dead = false;
        // a unit's queries, a piece of 16 bytes to a thread, and their scales
        uint4 query = make_uint4(0, 0, 0, 0);
        float mult = 0;
        auto loadQueries = [&](const TSegment &s) {
            const int chunk = s.Unit % p.HeadChunks, firstHead = s.Unit / p.HeadChunks * p.Group + chunk * PD_ROWS, rows = min(p.Group - chunk * PD_ROWS, PD_ROWS);
            const int r = tid / (D / 16), piece = tid % (D / 16);
            query = make_uint4(0, 0, 0, 0);
            if (r < rows) {
                query = *reinterpret_cast<const uint4 *>(p.Q.Row(s.Seq) + (firstHead + r) * D + piece * 16);
            }
            mult = p.QVecScale;
            if (tid < rows && p.QScale.Valid()) {
                mult = p.QScale.Row(s.Seq)[firstHead + tid];
            }
        };
        // as a K-major tile with the swizzle of the keys, once all score products with the unit's before are done
        auto storeQueries = [&](int n) {
            const int r = tid / (D / 16), piece = tid % (D / 16);
            if (r < PD_ROWS) {
                *reinterpret_cast<uint4 *>(qTile + r * D + (D == 128 ? piece ^ (r & 7) : piece ^ (r >> 1 & 3)) * 16) = query;
            }
            if (tid < PD_ROWS) {
                misc.Mult[n & 1][tid] = p.DotScale * mult;
            }
            FenceProxyAsync();
            MbarArrive(&misc.QReady);
        };
        loadQueries(walk.Segment(p));
        storeQueries(0);
        for (bool more = true; more; ++segments) {
            const TSegment seg = walk.Segment(p);
            const int head = seg.Unit / p.HeadChunks, chunk = seg.Unit % p.HeadChunks;
            const int firstHead = head * p.Group + chunk * PD_ROWS, rows = min(p.Group - chunk * PD_ROWS, PD_ROWS);
            more = walk.Next(p, seg);
            if (tid < PD_ROWS) {
                misc.Ref[tid] = misc.Top[tid] = PD_NO_REF;
            }
            float sum[HEADS], acc[HEADS];
#pragma unroll
            for (int h = 0; h < HEADS; ++h) {
                sum[h] = acc[h] = 0;
            }
            int sinceDrain = 0; // tiles whose products are in tensor memory
            // acc += what tensor memory has (the product with the weights of the tile before is done)
            auto drain = [&]() {
                TcFenceAfter();
#pragma unroll
                for (int b = 0; b < HB; ++b) {
                    uint32_t r[16];
                    TmemLd16(tmemOut + laneBase + b * 16, r);
                    TmemWaitLd();
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        if (E4M3) { // column 4 k + h: digit k
                            constexpr float STEP = 1 / PT_E4M3_STEP;
                            const float x = fmaf(STEP, fmaf(STEP, fmaf(STEP, __uint_as_float(r[12 + h]), __uint_as_float(r[8 + h])), __uint_as_float(r[4 + h])), __uint_as_float(r[h]));
                            acc[4 * b + h] = fmaf(x, 1 / PT_E4M3_UNIT, acc[4 * b + h]);
                        } else { // column 4 h + k: digit k, the lowest first
                            const float lo = fmaf(256.0f, (float)(int)r[4 * h + 1], (float)(int)r[4 * h]), hi = fmaf(256.0f, (float)(int)r[4 * h + 3], (float)(int)r[4 * h + 2]);
                            acc[4 * b + h] = fmaf(fmaf(65536.0f, hi, lo), 1 / PT_I8_UNIT, acc[4 * b + h]);
                        }
                    }
                }
                TcFenceBefore();
            };
            // the product with the weights of tile number n is done
            auto lastProduct = [&](int n) { return WaitBarA<true>(&misc.WFree[n % W_BUFS], (n / W_BUFS) & 1, abortFlag); };
            SoftAny(false); // Mult and Ref are there
            for (int tile = seg.TileBeg; tile < seg.TileEnd; ++tile, ++count) {
                const int buf = count & 1, stage = count % STAGES, wBuf = count % W_BUFS, key = tile * PT_KEYS + tid;
                const bool bringNext = more && tile == seg.TileEnd - 1;
                if (bringNext) {
                    loadQueries(walk.Segment(p));
                }
                if (!dead && !WaitBarA<true>(&misc.KeysFull[stage], (count / STAGES) & 1, abortFlag)) {
                    dead = true;
                    fail(kDevTimeoutMma);
                }
                const float ks = tileKeys[stage].KScale[tid], vs = tileKeys[stage].VScale[tid], bias = tileKeys[stage].Bias[tid];
                const bool valid = bias < INFINITY || bias != bias;
                const float edge = ReferenceEdge(vs, PT_EDGE);
                if (!dead && !WaitBarA<true>(&misc.SReady[buf], (count / 2) & 1, abortFlag)) {
                    dead = true;
                    fail(kDevTimeoutMma);
                }
                float z[16];
                __syncwarp();
                TcFenceAfter();
                {
                    uint32_t r[16];
                    TmemLd16(tmem + laneBase + buf * 16, r);
                    TmemWaitLd();
                    TcFenceBefore();
                    MbarArrive(&misc.SFree[buf]);
#pragma unroll
                    for (int h = 0; h < HEADS; ++h) {
                        z[h] = E4M3 ? __uint_as_float(r[h]) : (float)(int)r[h];
                    }
                }
                if (bringNext) {
                    storeQueries(segments + 1);
                }
                bool raise = false;
#pragma unroll
                for (int b = 0; b < HB; ++b) {
                    const float4 m4 = *reinterpret_cast<const float4 *>(&misc.Mult[segments & 1][4 * b]), r4 = *reinterpret_cast<const float4 *>(&misc.Ref[4 * b]);
                    const float mult[4] = {m4.x, m4.y, m4.z, m4.w}, ref[4] = {r4.x, r4.y, r4.z, r4.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float &y = z[4 * b + i];
                        y = valid ? fmaf(y * ks, mult[i], -bias) : -INFINITY;
                        raise |= y - ref[i] > edge;
                    }
                }
                if (p.Logits && key < seg.Keys.End) {
#pragma unroll
                    for (int h = 0; h < HEADS; ++h) {
                        if (h < rows) {
                            p.Logits[((size_t)seg.Seq * p.HeadCount + firstHead + h) * p.LogitRow + key] = z[h];
                        }
                    }
                }
                // the weights that had this place are used up
                if (!dead && count >= W_BUFS && !WaitBarA<true>(&misc.WFree[wBuf], (count / W_BUFS - 1) & 1, abortFlag)) {
                    dead = true;
                    fail(kDevTimeoutMma);
                }
                bool fresh = sinceDrain == 0;
                if (SoftAny(raise || dead || sinceDrain >= PT_DRAIN_TILES)) {
                    // new references: the largest z + log2 |vScale| of the tile's keys, not far below the highest so far; a tile without keys leaves them
#pragma unroll
                    for (int h = 0; h < HEADS; ++h) {
                        const int m = __reduce_max_sync(0xffffffffu, OrderedInt(z[h] != z[h] ? -INFINITY : z[h] - edge + PT_EDGE));
                        if (lane == 0) {
                            misc.Red[warp][h] = FromOrderedInt(m);
                        }
                    }
                    if (SoftAny(dead)) {
                        break;
                    }
                    if (sinceDrain > 0) {
                        if (!lastProduct(count - 1)) {
                            dead = true;
                            fail(kDevTimeoutMma);
                        }
                        __syncwarp();
                        drain();
                    }
                    float old = 0, ref = 0;
                    if (tid < HEADS) {
                        old = misc.Ref[tid];
                        const float most = ceilf(fmaxf(fmaxf(misc.Red[0][tid], misc.Red[1][tid]), fmaxf(misc.Red[2][tid], misc.Red[3][tid])));
                        const float top = fmaxf(misc.Top[tid], most);
                        ref = most == -INFINITY ? old : fmaxf(most, top - PT_SINK);
                        misc.Top[tid] = top;
                        misc.Ref[tid] = ref;
                        misc.Factor[tid] = WholeExp2(old - ref);
                    }
                    SoftAny(false);
#pragma unroll
                    for (int h = 0; h < HEADS; ++h) {
                        const float f = misc.Factor[h];
                        sum[h] *= f;
                        acc[h] *= f;
                    }
                    sinceDrain = 0;
                    fresh = true;
                }
#pragma unroll
                for (int b = 0; b < HB; ++b) {
                    const float4 r4 = *reinterpret_cast<const float4 *>(&misc.Ref[4 * b]);
                    const float ref[4] = {r4.x, r4.y, r4.z, r4.w};
                    float w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        w[i] = Exp2(z[4 * b + i] - ref[i]);
                        sum[4 * b + i] += w[i];
                    }
                    uint4 x;
                    if (E4M3) {
                        const float scale = vs * PT_E4M3_UNIT;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            w[i] *= scale;
                        }
                        uint32_t d[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t lo = TakeDigit(w[0], w[1]), hi = TakeDigit(w[2], w[3]);
                            d[k] = lo | hi << 16;
                        }
                        x = make_uint4(d[0], d[1], d[2], d[3]);
                    } else {
                        uint32_t d[4];
                        const float scale = vs * PT_I8_UNIT;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            d[i] = ((uint32_t)__float2int_rn(w[i] * scale) + 0x80808080u) ^ 0x80808080u; // signed digits of base 256
                        }
                        x = make_uint4(d[0], d[1], d[2], d[3]);
                    }
                    *reinterpret_cast<uint4 *>(wTile + wBuf * TL::W_BYTES + b * PT_KEYS * 16 + tid * 16) = x;
                }
                if (E4M3 && !valid) {
                    // what the slot holds may be NaN, which no weight of zero takes away
                    uint4 *v = reinterpret_cast<uint4 *>(smem + stage * 2 * TL::TILE_BYTES + TL::TILE_BYTES + tid * D);
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        v[i] = make_uint4(0, 0, 0, 0);
                    }
                }
                if (tid == 0) {
                    misc.Fresh[wBuf] = fresh;
                }
                FenceProxyAsync();
                MbarArrive(&misc.WReady[wBuf]);
                ++sinceDrain;
            }
            // the unit's last product
            if (!dead && !lastProduct(count - 1)) {
                dead = true;
                fail(kDevTimeoutMma);
            }
            if (SoftAny(dead)) {
                break;
            }
            drain();
            WarpSums(sum, lane);
            if ((lane & (32 / HEADS - 1)) == 0) {
                misc.Red[warp][HeadOfLane<HEADS>(lane)] = sum[0];
            }
            SoftAny(false);
            if (tid < rows) {
                float s = misc.Red[0][tid] + misc.Red[1][tid] + misc.Red[2][tid] + misc.Red[3][tid];
                const float m = misc.Ref[tid];
                if (seg.Whole) {
                    // the sink: weight 1 at logit 0
                    const float all = fmaxf(m, -60.0f), f = Exp2(m - all);
                    s = fmaf(f, s, Exp2(-all));
                    misc.Factor[tid] = f / s;
                    if (p.Lse) {
                        p.Lse[(size_t)seg.Seq * p.HeadCount + firstHead + tid] = all + Log2(s);
                    }
                } else {
                    float *dst = PartialRecord(p, D, blockIdx.x, seg.Seq, seg.Unit, tid);
                    dst[D] = m;
                    dst[D + 1] = s;
                }
            }
            SoftAny(false);
            if (hasDim) {
                if (seg.Whole) {
#pragma unroll
                    for (int h = 0; h < HEADS; ++h) {
                        if (h < rows) {
                            StoreFromFloat(p.Out.Row(seg.Seq), (firstHead + h) * D + dim, p.OutDtype, acc[h] * misc.Factor[h]);
                        }
                    }
                } else {
                    float *dst = PartialRecord(p, D, blockIdx.x, seg.Seq, seg.Unit, 0) + dim;
#pragma unroll
                    for (int h = 0; h < HEADS; ++h) {
                        if (h < rows) {
                            dst[h * (D + 4)] = acc[h];
                        }
                    }
                }
            }
            SoftAny(false); // Red, Ref and Factor have been read
        }
    }
    TcFenceBefore();
    __syncthreads();
    if (warp == PT_MMA_WARP) {
        TcFenceAfter();
        TmemDealloc(tmem, PT_TMEM_COLS);
    }
}

template <int D, bool E4M3>
static const void *PickBlocks(int rows, size_t *smem, int *perSm)
{
    if (rows <= 4) {
        *smem = TTcLayout<D, 1>::BYTES;
        *perSm = TTcLayout<D, 1>::CTAS;
        return (const void *)PagedRangeKernel<D, E4M3, 1>;
    }
    if (rows <= 8) {
        *smem = TTcLayout<D, 2>::BYTES;
        *perSm = TTcLayout<D, 2>::CTAS;
        return (const void *)PagedRangeKernel<D, E4M3, 2>;
    }
    *smem = TTcLayout<D, 4>::BYTES;
    *perSm = TTcLayout<D, 4>::CTAS;
    return (const void *)PagedRangeKernel<D, E4M3, 4>;
}

int LaunchPagedRanges(const TPagedDecodeParams &p, const tsa_paged_kv *kv, int headDim, bool e4m3, long long tilesMax, unsigned *ctas, cudaStream_t stream)
{
    const long long slots = ((long long)kv->page_count * kv->kv_heads) << p.C.PageShift;
    if (slots > 0x7fffff00) {
        return Fail(TSA_UNSUPPORTED, "tsa_paged_decode: %d pages of %d slots and %d key heads are more than 2^31 rows", kv->page_count, kv->page_size, kv->kv_heads);
    }
    const int box = kv->page_size < PT_KEYS ? kv->page_size : PT_KEYS;
    CUtensorMap tmK, tmV;
    const tsa_ptr2d k = {kv->k, headDim, headDim, (int)slots}, v = {kv->v, headDim, headDim, (int)slots};
    int rc = MakeTileMapEx(&tmK, k, 1, headDim, box, "paged keys");
    if (rc == TSA_OK) {
        rc = MakeTileMapEx(&tmV, v, 1, headDim, box, "paged values");
    }
    if (rc != TSA_OK) {
        return rc;
    }
    size_t smem = 0;
    int perSm = 0;
    const void *kern = headDim == 128 ? (e4m3 ? PickBlocks<128, true>(p.Rows, &smem, &perSm) : PickBlocks<128, false>(p.Rows, &smem, &perSm))
                                      : (e4m3 ? PickBlocks<64, true>(p.Rows, &smem, &perSm) : PickBlocks<64, false>(p.Rows, &smem, &perSm));
    int dev = 0, sms = 0;
    rc = CheckCuda(cudaGetDevice(&dev), "cudaGetDevice");
    if (rc == TSA_OK) {
        rc = CheckCuda(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev), "cudaDeviceGetAttribute");
    }
    if (rc == TSA_OK) {
        rc = CheckCuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "cudaFuncSetAttribute");
    }
    if (rc != TSA_OK) {
        return rc;
    }
    const long long total = tilesMax * p.NSeq * kv->kv_heads * p.HeadChunks;
    *ctas = (unsigned)(total < perSm * sms ? total : perSm * sms);
    *ctas = *ctas < PD_MAX_CTAS ? *ctas : PD_MAX_CTAS;
    TPagedDecodeParams copy = p;
    void *args[] = {&tmK, &tmV, &copy};
    // Three CTAs to an SM find no place on some while the kernel before is still there, and the ones left over run alone at the end: with eight
    // tiles each or more they rather come when it has gone (64 dimensions, 512 key heads of 2000 .. 6000 slots: 66 us, and 57.6 this way; five tiles each,
    // 64 of 4100: 13.4 and 14.8; two CTAs to an SM, 128 dimensions, 8 of 100000 .. 131072: 49.3 and 51.5)
    if (perSm > 2 && total >= 8ll * *ctas) {
        return CheckCuda(cudaLaunchKernel(kern, dim3(*ctas), dim3(PT_THREADS), args, smem, stream), "tsa_paged_decode launch");
    }
    return CheckCuda(LaunchPdl(kern, dim3(*ctas), dim3(PT_THREADS), smem, stream, args), "tsa_paged_decode launch");
}

} // namespace tsa

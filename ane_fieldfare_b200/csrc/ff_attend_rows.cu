// Attention of up to 16 columns a key/value head (decode steps, short verify blocks) over the paged INT4 cache.
//
// The columns of a request's key/value head are its rows times the query heads that share the head; they stand in
// tiles of 8 NT.  A unit of work is one (request, key/value head, column tile); its keys are tiles of 64, and all
// units' tiles end to end are cut into equal runs, one per CTA, so that one long request fills the GPU and a ragged
// batch leaves no SM with more than another.  A unit that several CTAs share is joined by whichever of them ends last,
// in the CTAs' order: the same bits every time, and nothing waits.
//
// In a CTA one warp copies (TMA boxes of codes, bulk copies of scale words, a ring of tiles); four warps take 32 keys of
// every second tile each, with a maximum, sum and output of their own, joined at the end of a unit.  Per 16 keys:
//   S = K q   codes as they lie are the A operand: a nibble masked in place IS an f16, the subnormal code * 2^-24 or
//             * 2^-20, exact, so a word of eight codes costs five instructions.  q is B, in f16 at a power of two of its
//             own (bf16 fits f16's 11 bits; what lies 2^-28 below the largest is lost).  Per group of 64 the 32-bit sum
//             takes the group's scale, and the bias times the group's sum of q is added, in fp32.
//   O += V p  codes of two keys are merged by a byte permute; the value scale goes into p (f16, one rounding more), at a
//             power of two E that keeps the largest scale and bias of the unit so far within f16 (raised like the
//             running maximum); one more MMA adds up p * bias per group and p itself.
// Logits are then exact but for 32-bit sums.  A weight is rounded to 11 bits once, for sum and output alike; times the value scale it
// would be rounded again, so that the codes' and the biases' part of a value that is near zero would not cancel: what that
// rounding leaves goes through a second product (up to four columns: through the four columns that a tile of eight has to spare).
// A weight below 2^-24 of the largest of its warp's keys so far is lost, and what of a value is below 2^-31 of the largest value so far.
//
// Bound by the cache's bytes and by latency.  131072 keys of 8 heads of 128 (151 MB) take 46.8 us, 3.2 TB/s or 49 % of a copy's
// rate; with the arithmetic left out 33 us.  A warp executes about 610 instructions for 32 keys of 128, all of the kernel's counted.  64
// ragged requests (261 MB) take 76.5 us, 3.4 TB/s, at 46 % of the issue slots, and 53 us with the arithmetic left out.  Three CTAs an SM
// with fewer registers a thread: 131072 keys 48.4 us where two took 44.3, ragged 73.4 and 73.1.  2000 keys of 8 heads of 256 are 14.1 us of
// waits one after another (in a timeline of 13.5: look-up of the requests 1.0, queries 1.7, tiles 3.4, joins in the CTA 1 and of the
// parts 2; the checks of lengths and row starts came behind it).
// Registers: none spill at 64 values a head; at 128, 240 bytes with more than 8 columns; at 256, 144 bytes with up to 4 columns, 128
// with up to 8 and 532 with more, which also leave room for one CTA an SM alone.
#include <algorithm>
#include <string>

#include "ff_attention_device.cuh"

namespace ff {

namespace {

constexpr int kConsumers = 4;                      // warps that compute: two a tile, 32 keys each
constexpr int kRowsThreads = 32 * (kConsumers + 1);
constexpr uint32_t kWaitLimit = 1u << 20;
constexpr uint32_t kUnitCost = 8;                 // tiles' time that a unit takes besides its tiles
static_assert(kTileKeys == 64 && kConsumers == 4, "two warps a tile, 32 keys each");

struct RowsArgs {
    AttendArgs a;
    float *partials;      // [2 CTAs][columns][DIM]
    float2 *stats;        // [2 CTAs][columns] maximum (log2), sum
    uint32_t *arrived;    // [3][CTAs], zero between launches: of a unit, of its first group of parts, of another group
    uint32_t pageShift, pieceShift;  // log2 of a page's tokens and of the keys of a tile on one page
};

__host__ __device__ constexpr uint32_t rows_stage_bytes(int dim) { return (kTileKeys * (dim + dim / 8) + 1023u) & ~1023u; }
__host__ __device__ constexpr uint32_t rows_stages(int dim) { return dim == 256 ? 4u : 6u; }
__host__ __device__ constexpr uint32_t rows_smem(int dim, int nt) {
    return 1024u + rows_stages(dim) * rows_stage_bytes(dim) + 2u * 8u * nt * (dim + 4) * 4u;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the first product of a sum
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// a * b - c
__device__ __forceinline__ uint32_t residual_f16x2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("{\n.reg .b32 n;\nneg.f16x2 n, %3;\nfma.rn.f16x2 %0, %1, %2, n;\n}" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ uint32_t max_f16x2(uint32_t a, uint32_t b) {  // NaN if either is
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// nibbles u and u + 4 of a word as an f16 pair: codes * 2^-24 (u even) or * 2^-20
template <int U>
__device__ __forceinline__ uint32_t nibbles(uint32_t w, uint32_t upper) {
    return (U < 2 ? w : upper) & (U % 2 ? 0x00F000F0u : 0x000F000Fu);
}

// The rest of a wait whose first look found nothing: up to a limit, or until another warp of the CTA has given up.
__device__ __noinline__ void wait_rows(uint32_t bar, uint32_t parity, volatile uint32_t *abortFlag) {
#pragma unroll 1
    for (uint32_t i = 0; i < kWaitLimit; ++i) {
        if ((i & 255u) == 0u && *abortFlag) return;
        if (mbar_try_wait(bar, parity)) return;
    }
    *abortFlag = 1u;
}

// One request as the kernel sees it.
struct RowsRequest {
    uint32_t firstRow, rows, tilesSink, lowTile, tiles, columnTiles;
    int length, p0;  // p0: position of its first row
};

// MMA row r (0..7) of eight keys: the key it stands for.  A permutation with which the eight lanes a quarter reads codes
// of fall into different banks under the copies' swizzle.
template <int DIM>
__device__ __forceinline__ uint32_t key_of_row(uint32_t r) {
    if (DIM == 256) return r;
    const uint32_t t = r >> 1, odd = r & 1u;
    return DIM == 128 ? (t & 1u) | (odd << 1) | ((t & 2u) << 1) : t | (odd << 2);
}
template <int DIM, int NT, bool SPLIT>
__global__ void __launch_bounds__(kRowsThreads, DIM * NT <= 256 ? 2 : 1) k_attend_rows(const __grid_constant__ CUtensorMap mapCodes, const __grid_constant__ CUtensorMap mapWords, const RowsArgs args) {
    constexpr int NG = DIM / 64, CB = DIM / 2, WB = NG * 4;
    constexpr uint32_t kStage = rows_stage_bytes(DIM), kStages = rows_stages(DIM), kColumns = SPLIT ? 4 : 8 * NT;
    static_assert(!SPLIT || NT == 1, "four columns, each twice");
    constexpr uint32_t kKeyWords = kTileKeys * CB * 2;
    extern __shared__ uint8_t rowsSmem[];
    __shared__ __align__(8) uint64_t barriers[2 * 6];
    __shared__ uint32_t first[kRowsThreads + 1], warpSums[kConsumers + 1], holes[6];
    __shared__ float2 joinStats[kConsumers][kColumns];
    __shared__ float joinBias[kConsumers][NG][kColumns];
    __shared__ uint32_t lastPart;
    __shared__ volatile uint32_t abortFlag;  // a wait was given up: nothing more is copied, what there is to multiply and join goes on
    __shared__ RowsRequest known[kRowsThreads];
    const AttendArgs &a = args.a;
    const uint32_t tid = threadIdx.x, warp = (uint32_t)warp_index(), lane = tid & 31u;
    const uint32_t ring = (sm_addr(rowsSmem) + 1023u) & ~1023u;
    float *joined = reinterpret_cast<float *>(rowsSmem + (ring - sm_addr(rowsSmem)) + kStages * kStage);
    const uint32_t group = a.heads / a.kvHeads;
    const uint32_t barFull = sm_addr(barriers), barEmpty = barFull + 8 * kStages;
    if (tid == 0) {
        abortFlag = 0;
        for (uint32_t s = 0; s < kStages; ++s) {
            bar_init(barFull + 8 * s, 1);
            bar_init(barEmpty + 8 * s, kConsumers / 2);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_enter();

    // ---- the plan: how many tiles each request is, and this CTA's run of them ----
    auto look_up = [&](uint32_t r) {
        RowsRequest q{};
        const uint32_t begin = min(__ldg(a.rowStart + r), a.tokens), end = min(__ldg(a.rowStart + r + 1), a.tokens);
        const uint32_t rows = end > begin ? end - begin : 0u;
        q.firstRow = begin;
        q.length = (int)min(__ldg(a.lengths + r), 0x7FFFFFFFu);
        q.p0 = q.length - (int)rows;
        q.rows = min(rows, a.maxRows);
        if (q.rows == 0) return q;
        q.columnTiles = (q.rows * group + kColumns - 1) / kColumns;
        const uint32_t last = (uint32_t)max(0, q.p0 + (int)q.rows), ends = (min(last, a.tableKeys) + kTileKeys - 1) / kTileKeys;
        if (a.window) {
            const uint32_t low = (uint32_t)max((long long)0, (long long)q.p0 - (long long)a.window + 1);
            q.lowTile = min(low / kTileKeys, ends);
            q.tilesSink = min((uint32_t)(((unsigned long long)a.sinks + kTileKeys - 1) / kTileKeys), q.lowTile);
        }
        q.tiles = max(1u, q.tilesSink + ends - q.lowTile);  // (a request without keys: one tile that nobody sees)
        return q;
    };
    // A unit costs its tiles and kUnitCost more: its queries, joins and output take as long.  (Cut by tiles alone, the CTAs with the
    // short requests of a ragged batch took 94 us where the others took 62.  kUnitCost 1, 3, 6, 8, 10, 14: ragged 90, 81, 72, 73,
    // 74, 78 us, 4 x 16 rows in a window 42, 39, 36, 35, 37, 37; 1 and 3 with CTAs of two tiles or more, the others of three.)
    auto unit_cost = [](const RowsRequest &q) { return q.rows ? q.tiles + kUnitCost : 0u; };
    const uint32_t run = (a.requests + kRowsThreads - 1) / kRowsThreads;
    auto request_of = [&](uint32_t r) { return run == 1 ? known[r] : look_up(r); };  // (a batch of up to 160 is looked up once)
    const uint32_t r0 = min(tid * run, a.requests), r1 = min(r0 + run, a.requests);
    // rowStart goes back, to rows that several requests would write: such a call is refused like one with too much work
    auto goes_back = [&](uint32_t r) { return __ldg(a.rowStart + r + 1) < __ldg(a.rowStart + r); };
    uint32_t sum = 0;
    for (uint32_t r = r0; r < r1; ++r) {
        const RowsRequest q = look_up(r);
        if (run == 1) known[r] = q;
        if (q.rows && q.p0 + (int)q.rows > 0 && (uint32_t)(q.p0 + (int)q.rows) > a.tableKeys) *a.errorFlag = kFlagTableRow;  // (what the row has no room for is not walked)
        sum = add_work(sum, work_of(unit_cost(q), q.columnTiles * a.kvHeads));
        if (goes_back(r)) sum = kTooMuch;
    }
    uint32_t scan = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, scan, d);
        if (lane >= (uint32_t)d) scan = add_work(scan, v);
    }
    if (lane == 31u) warpSums[warp] = scan;
    __syncthreads();
    uint32_t before = 0, total = 0;
#pragma unroll
    for (uint32_t w = 0; w <= (uint32_t)kConsumers; ++w) {
        if (w < warp) before += warpSums[w];
        total = add_work(total, warpSums[w]);
    }
    const bool refused = total == kTooMuch;  // (the places of units are nothing then)
    first[tid] = before + scan - sum;
    if (tid == 0) first[kRowsThreads] = total;
    __syncthreads();

    // rows that no unit writes: behind the last request's, and past maxRows
    {
        const uint32_t covered = a.requests && !refused ? min(__ldg(a.rowStart + a.requests), a.tokens) : 0u;
        const uint32_t perRow = a.heads * DIM / 8;
        for (uint32_t row = covered + blockIdx.x; row < a.tokens; row += gridDim.x)
            for (uint32_t i = tid; i < perRow; i += kRowsThreads) *reinterpret_cast<uint4 *>(a.out + (size_t)row * a.outStride + i * 8) = make_uint4(0u, 0u, 0u, 0u);
        if (blockIdx.x == 0) {
            if (tid == 0 && refused) *a.errorFlag = kFlagWork;
            __syncthreads();
            if (tid == 0 && a.requests && __ldg(a.rowStart + a.requests) > a.tokens) *a.errorFlag = kFlagRows;
            for (uint32_t r = r0; r < r1; ++r) {
                if (goes_back(r)) *a.errorFlag = kFlagRows;
                if (refused) continue;
                const uint32_t begin = min(__ldg(a.rowStart + r), a.tokens), end = min(__ldg(a.rowStart + r + 1), a.tokens);
                for (uint32_t row = begin + a.maxRows; row < end; ++row) {
                    *a.errorFlag = kFlagRows;
                    for (uint32_t i = 0; i < perRow; ++i) *reinterpret_cast<uint4 *>(a.out + (size_t)row * a.outStride + i * 8) = make_uint4(0u, 0u, 0u, 0u);
                }
            }
        }
    }
    if (total == 0 || refused) return;
    const uint32_t ctas = min(gridDim.x, max(1u, total / 3u)), cta = blockIdx.x;
    if (cta >= ctas) return;
    auto start_of = [&](uint32_t c) { return (uint32_t)((unsigned long long)c * total / ctas); };
    auto cta_of = [&](uint32_t x) { return (uint32_t)((((unsigned long long)x + 1) * ctas - 1) / total); };
    const uint32_t begin = start_of(cta), end = start_of(cta + 1);

    // Where the run stands: a request's unit, whose tile i stands at x = first + kUnitCost + i; and the tiles of it that are
    // this CTA's.
    struct Walk {
        uint32_t r, unit, first;
        RowsRequest q;
        uint32_t t0, count, head, column0;
    };
    auto take = [&](Walk &w) {
        const uint32_t tile0 = w.first + kUnitCost;
        w.t0 = begin > tile0 ? min(begin - tile0, w.q.tiles) : 0u;
        w.count = (end > tile0 ? min(end - tile0, w.q.tiles) : 0u) - w.t0;
        w.head = w.unit / w.q.columnTiles;
        w.column0 = w.unit % w.q.columnTiles * kColumns;
    };
    auto locate = [&](uint32_t x) {
        uint32_t low = 0, high = kRowsThreads;
        while (high - low > 1) {
            const uint32_t mid = (low + high) >> 1;
            if (first[mid] <= x) low = mid;
            else high = mid;
        }
        Walk w;
        uint32_t n = x - first[low];
        for (w.r = low * run;; ++w.r) {
            w.q = request_of(w.r);
            const uint32_t mine = unit_cost(w.q) * w.q.columnTiles * a.kvHeads;
            if (n < mine) break;
            n -= mine;
        }
        w.unit = n / unit_cost(w.q);
        w.first = x - n % unit_cost(w.q);
        take(w);
        return w;
    };
    // the unit behind; false past the run's end
    auto next_unit = [&](Walk &w) {
        w.first += unit_cost(w.q);
        if (w.first >= end) return false;
        if (++w.unit == w.q.columnTiles * a.kvHeads) {
            w.unit = 0;
            do {
                w.q = request_of(++w.r);
            } while (w.q.rows == 0);
        }
        take(w);
        return true;
    };

    if (warp == (uint32_t)kConsumers) {
        // ---------------- copies ----------------
        // A lane holds the page of one piece (the keys of a tile on one page): 32 pieces at a time, the next 32 in flight.
        // The warp runs as one and an elected lane issues: a copy in a branch that lanes take apart costs several hundred cycles,
        // its operands go to the uniform registers by a loop over the lanes.
        const uint32_t pieces = kTileKeys >> args.pieceShift, perTileShift = 6u - args.pieceShift;
        const uint32_t tilesPer = 32u >> perTileShift;  // tiles whose pieces a warp holds
        const uint32_t pieceCodes = 2u * CB << args.pieceShift, pieceWords = 2u * WB << args.pieceShift;
        uint32_t stage = 0, phase = 0;
        bool ok = true;
        Walk w = locate(begin);
        do {
            const uint32_t t0 = w.t0, count = w.count, head = w.head;
            if (count == 0) continue;
            const int keysEnd = w.q.p0 + (int)w.q.rows;
            auto key_at = [&](uint32_t t) { return (t < w.q.tilesSink ? t : w.q.lowTile + t - w.q.tilesSink) * kTileKeys; };
            auto page_of = [&](uint32_t base) {
                const uint32_t t = base + (lane >> perTileShift);
                uint32_t page = FF_NO_PAGE;
                if (t < t0 + count) {
                    const uint32_t key = key_at(t) + ((lane & (pieces - 1u)) << args.pieceShift);
                    if ((int)key < keysEnd) {
                        const uint32_t index = key >> args.pageShift;
                        if (index < a.tableStride) page = __ldg(a.blockTable + (size_t)w.r * a.tableStride + index);
                        else *a.errorFlag = kFlagTableRow;
                        if (page >= a.pageCount && index < a.tableStride) *a.errorFlag = kFlagPage;
                    }
                }
                return page;
            };
            uint32_t pagesNext = page_of(t0);
            for (uint32_t t = t0; t < t0 + count && ok; t += tilesPer) {
                const uint32_t pagesNow = pagesNext;
                pagesNext = page_of(t + tilesPer);
                const uint32_t many = min(tilesPer, t0 + count - t);
                for (uint32_t i = 0; i < many; ++i) {
                    const uint32_t mine = __shfl_sync(0xFFFFFFFFu, pagesNow, (i << perTileShift) + (lane & (pieces - 1u)));
                    const uint32_t lives = __ballot_sync(0xFFFFFFFFu, lane < pieces && mine < a.pageCount);
                    if (!mbar_try_wait(barEmpty + 8 * stage, phase ^ 1u)) wait_rows(barEmpty + 8 * stage, phase ^ 1u, &abortFlag);
                    if (!(ok = __all_sync(0xFFFFFFFFu, abortFlag == 0u))) break;  // (a stage may still wait for its copies)
                    const uint32_t bar = barFull + 8 * stage, base = ring + stage * kStage, inTile = key_at(t + i) & (a.page.pageTokens - 1u);
                    if (elect_one()) {
                        holes[stage] = ~lives;
                        bar_expect(bar, (uint32_t)__popc(lives) * (pieceCodes + pieceWords));
                    }
                    for (uint32_t p = 0; p < pieces; ++p) {
                        const uint32_t block = __shfl_sync(0xFFFFFFFFu, mine, p) * a.kvHeads + head, at = (inTile + (p << args.pieceShift)) & (a.page.pageTokens - 1u);
                        if ((lives >> p & 1u) && elect_one()) {
                            tma_load_4d(base + p * pieceCodes, &mapCodes, 0, (int)at, 0, (int)block, bar);
                            tma_load_3d(base + kKeyWords + p * pieceWords, &mapWords, (int)(at * NG), 0, (int)block, bar);
                        }
                    }
                    if (++stage == kStages) stage = 0, phase ^= 1u;
                }
            }
        } while (ok && next_unit(w));
        // also where a consumer gave up: no copy is in flight when the CTA ends
        for (uint32_t s = 0; s < kStages; ++s) {
            const uint32_t parity = s < stage ? phase : phase ^ 1u;
#pragma unroll 1
            for (uint32_t i = 0; i < kWaitLimit && !mbar_try_wait(barFull + 8 * s, parity); ++i) __nanosleep(40);
        }
        if (lane == 0 && abortFlag) *a.errorFlag = kFlagWait;
        return;
    }

    // ---------------- 32 keys of every second tile ----------------
    const uint32_t g = lane >> 2, t = lane & 3u;
    // A stage: [piece][keys, values][its keys][codes], then [piece][keys, values][its keys][words].  Warps 0 and 1 take half of
    // every second tile each, warps 2 and 3 of the others: 32 keys at a time as two subtiles of 16, for whose loads and products
    // there is then other work to do, and one round of everything that is done once.
    const uint32_t warpKey = 32 * (warp & 1u);
    const uint32_t keyA = key_of_row<DIM>(g);  // the S fragments' rows: keys keyA and keyA + 8 of a subtile
    const uint32_t vStep = 1u << args.pieceShift;
    uint32_t subRow[2];  // first row of a subtile's keys: a piece's values lie behind its keys
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
        const uint32_t key = warpKey + 16 * sub;
        subRow[sub] = key + ((key >> args.pieceShift) << args.pieceShift);
    }
    uint32_t kOff[NG], vOff[2][NG];  // in a subtile, by group; the P fragments' keys 2t and 2t + 1; those + 8 follow
#pragma unroll
    for (int G = 0; G < NG; ++G) {
        kOff[G] = keyA * CB + ((G * 32 + t * 8) ^ chunk_flip<DIM>(keyA));
#pragma unroll
        for (int i = 0; i < 2; ++i) vOff[i][G] = (key_of_row<DIM>(2 * t + i) + vStep) * CB + ((G * 32 + g * 4) ^ chunk_flip<DIM>(key_of_row<DIM>(2 * t + i)));
    }
    // Value scales are converted once, a pair of keys (rows 2j, 2j + 1 of a subtile) and group to a lane, and handed round:
    // lane (and element e) = subtile * 8 + j, group = 2 e + lane / 16 (dim 64: lanes from 16 on repeat)
    constexpr int kPairs = NG == 4 ? 2 : 1;
    const uint32_t pairSub = (lane >> 3) & 1u, pairRow = 2 * (lane & 7u), pairGroup = NG == 1 ? 0u : lane >> 4;
    uint32_t pairKey[2];  // in the warp's 32
#pragma unroll
    for (int i = 0; i < 2; ++i) pairKey[i] = 16 * pairSub + (pairRow & 8u) + key_of_row<DIM>((pairRow & 7u) + i);
    const uint32_t pairWord = (subRow[0] + vStep + (pairSub ? subRow[1] - subRow[0] - 16 : 0u)) * WB + pairGroup * 4;  // + pairKey * WB
    Walk w = locate(begin);
    uint32_t n0 = 0;  // tiles so far: they are counted over the CTA's run, for their stage and the warps that take them
    do {
        const uint32_t t0 = w.t0, count = w.count, head = w.head, column0 = w.column0, unitTiles = w.q.tiles;
        if (count == 0) continue;  // (the run begins or ends in front of the unit's first tile)
        const uint32_t columns = w.q.rows * group;
        // queries: f16 at a power of two of the column's largest value
        uint32_t qf[NG][4][NT][2];
        float qSum[NG][NT][2], toLog2[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint32_t column = column0 + 8 * n + (SPLIT ? g & 3u : g), row = column / group;
            const bool there = column < columns;
            const uint16_t *src = a.q + (size_t)(w.q.firstRow + row) * a.qStride + (head * group + column % group) * DIM + 16 * t;
            uint4 v[NG][2];
            uint32_t largest = 0;
#pragma unroll
            for (int G = 0; G < NG; ++G)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    v[G][i] = there ? __ldg(reinterpret_cast<const uint4 *>(src + 64 * G + 8 * i)) : make_uint4(0u, 0u, 0u, 0u);
                    largest = __vmaxu2(largest, __vmaxu2(__vmaxu2(v[G][i].x & 0x7FFF7FFFu, v[G][i].y & 0x7FFF7FFFu), __vmaxu2(v[G][i].z & 0x7FFF7FFFu, v[G][i].w & 0x7FFF7FFFu)));
                }
            uint32_t exponent = max(largest & 0xFFFFu, largest >> 16) >> 7;
            exponent = max(exponent, __shfl_xor_sync(0xFFFFFFFFu, exponent, 1));
            exponent = max(exponent, __shfl_xor_sync(0xFFFFFFFFu, exponent, 2));
            exponent = max(exponent, 13u);
            const float down = __uint_as_float((267u - exponent) << 23);  // 2^(13 - (exponent - 127)): the largest is 2^13 .. 2^14
            float mine[NG];
#pragma unroll
            for (int G = 0; G < NG; ++G) {
                float f[16];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t u[4] = {v[G][i].x, v[G][i].y, v[G][i].z, v[G][i].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) f[8 * i + 2 * j] = low16(u[j]) * down, f[8 * i + 2 * j + 1] = high16(u[j]) * down;
                }
                mine[G] = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) mine[G] += f[i];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float odd = u % 2 ? 0.0625f : 1.0f;
                    qf[G][u][n][0] = pack_f16(f[u] * odd, f[u + 4] * odd);
                    qf[G][u][n][1] = pack_f16(f[8 + u] * odd, f[12 + u] * odd);
                }
                mine[G] += __shfl_xor_sync(0xFFFFFFFFu, mine[G], 1);
                mine[G] += __shfl_xor_sync(0xFFFFFFFFu, mine[G], 2);
            }
            // the S fragments' columns are 2t and 2t + 1
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const uint32_t from = (2 * t + c) * 4;
#pragma unroll
                for (int G = 0; G < NG; ++G) qSum[G][n][c] = __shfl_sync(0xFFFFFFFFu, mine[G], from) * 0x1p-24f;
                // q = f16 * 2^(exponent - 140), the codes are 2^-24 of theirs
                toLog2[n][c] = logit_factor(a.scale, (int)__shfl_sync(0xFFFFFFFFu, exponent, from) - 116);
            }
        }

        float o[NG][4][NT][4], extra[NT][4], top[NT][2];
        int E = -120;
        float toE = power_of_two(120);  // 2^-E
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int G = 0; G < NG; ++G)
#pragma unroll
                for (int v = 0; v < 4; ++v)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[G][v][n][i] = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) extra[n][i] = 0.0f;
            top[n][0] = top[n][1] = kNone;
        }
        const int pFirst = w.q.p0 + (int)(column0 / group), pLast = w.q.p0 + (int)((min(columns, column0 + kColumns) - 1) / group);

        for (uint32_t i = t0 + ((n0 ^ (warp >> 1)) & 1u); i < t0 + count; i += 2) {
            const uint32_t number = n0 + i - t0, stage = number % kStages, phase = number / kStages & 1u;
            const uint32_t tileKey = (i < w.q.tilesSink ? i : w.q.lowTile + i - w.q.tilesSink) * kTileKeys;
            const int j0 = (int)(tileKey + warpKey);
            const uint32_t base = ring + stage * kStage;
            if (!mbar_try_wait(barFull + 8 * stage, phase)) wait_rows(barFull + 8 * stage, phase, &abortFlag);
            __syncwarp();
            const uint32_t gone = holes[stage], hole0 = gone >> (warpKey >> args.pieceShift) & 1u, hole1 = gone >> ((warpKey + 16) >> args.pieceShift) & 1u;
            // keys that not every row of the tile sees
            const bool careful = (hole0 | hole1) || j0 + 31 > pFirst || (a.window && (long long)j0 <= (long long)pLast - a.window && (uint32_t)j0 + 32u > a.sinks);
            auto sees = [&](int key, int p) {
                return key <= p && (!a.window || (long long)key > (long long)p - a.window || (uint32_t)key < a.sinks) && !((uint32_t)(key - j0) < 16u ? hole0 : hole1);
            };

            // ---- value scales as f16 pairs of keys, at 2^-E ----
            uint32_t pairs[kPairs][2];
#pragma unroll
            for (int e = 0; e < kPairs; ++e)
#pragma unroll
                for (int k = 0; k < 2; ++k) pairs[e][k] = lds32(base + kKeyWords + pairWord + pairKey[k] * WB + 8 * e);
            if (careful) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int key = j0 + (int)pairKey[k], p = max(key, pFirst);  // of the rows that may see it, the one whose window goes back furthest
                    if (p > pLast || !sees(key, p))
#pragma unroll
                        for (int e = 0; e < kPairs; ++e) pairs[e][k] = 0u;
                }
            }
            uint32_t pairScale[kPairs], pairBias[kPairs];
            auto convert = [&] {
                const float f = toE;
                uint32_t most = 0;
#pragma unroll
                for (int e = 0; e < kPairs; ++e) {
                    pairScale[e] = pack_f16(low16(pairs[e][0]) * f, low16(pairs[e][1]) * f);
                    pairBias[e] = pack_f16(high16(pairs[e][0]) * f, high16(pairs[e][1]) * f);
                    most = max_f16x2(most, max_f16x2(pairScale[e], pairBias[e] & 0x7FFF7FFFu));
                }
                return __vmaxu2(most, 0x54005400u) != 0x54005400u;  // beyond 2^6, or NaN
            };
            uint32_t broken[2] = {0u, 0u};  // lanes whose pair's first, second key has a value that is no number
            if (__any_sync(0xFFFFFFFFu, convert())) {
                uint32_t most = 0;
#pragma unroll
                for (int e = 0; e < kPairs; ++e)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const bool bad = is_broken(pairs[e][k]);
                        broken[k] |= __ballot_sync(0xFFFFFFFFu, bad);
                        if (bad) pairs[e][k] = 0u;
                        most = max(most, word_exponent(pairs[e][k]));
                    }
                most = __reduce_max_sync(0xFFFFFFFFu, most);
                const int raised = min(max((int)most - 127 - 5, E), 120);
                if (raised > E) {
                    const float f = power_of_two(E - raised);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int G = 0; G < NG; ++G)
#pragma unroll
                            for (int v = 0; v < 4; ++v)
#pragma unroll
                                for (int k = 0; k < 4; ++k) o[G][v][n][k] *= f;
                        extra[n][0] *= f;
                        extra[n][1] *= f;
                    }
                    E = raised;
                    toE = power_of_two(-E);
                }
                convert();
            }

            // ---- logits ----
            float s[2][NT][4];
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                uint32_t kWords[2][NG];
                lds_words<NG>(base + kKeyWords + (subRow[sub] + keyA) * WB, kWords[0]);
                lds_words<NG>(base + kKeyWords + (subRow[sub] + keyA + 8) * WB, kWords[1]);
                const uint32_t row = base + subRow[sub] * CB;
#pragma unroll
                for (int n = 0; n < NT; ++n) s[sub][n][0] = s[sub][n][1] = s[sub][n][2] = s[sub][n][3] = 0.0f;
#pragma unroll
                for (int G = 0; G < NG; ++G) {
                    const uint2 wa = lds64(row + kOff[G]), wb = lds64(row + kOff[G] + 8 * CB);
                    const uint32_t ax = wa.x >> 8, ay = wa.y >> 8, bx = wb.x >> 8, by = wb.y >> 8;
                    float acc[NT][4];
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_f16_first(acc[n], nibbles<0>(wa.x, ax), nibbles<0>(wb.x, bx), nibbles<0>(wa.y, ay), nibbles<0>(wb.y, by), qf[G][0][n][0], qf[G][0][n][1]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_f16(acc[n], nibbles<1>(wa.x, ax), nibbles<1>(wb.x, bx), nibbles<1>(wa.y, ay), nibbles<1>(wb.y, by), qf[G][1][n][0], qf[G][1][n][1]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_f16(acc[n], nibbles<2>(wa.x, ax), nibbles<2>(wb.x, bx), nibbles<2>(wa.y, ay), nibbles<2>(wb.y, by), qf[G][2][n][0], qf[G][2][n][1]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_f16(acc[n], nibbles<3>(wa.x, ax), nibbles<3>(wb.x, bx), nibbles<3>(wa.y, ay), nibbles<3>(wb.y, by), qf[G][3][n][0], qf[G][3][n][1]);
                    const float sa = low16(kWords[0][G]), ba = high16(kWords[0][G]), sb = low16(kWords[1][G]), bb = high16(kWords[1][G]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        s[sub][n][0] = fmaf(sa, acc[n][0], fmaf(ba, qSum[G][n][0], s[sub][n][0]));
                        s[sub][n][1] = fmaf(sa, acc[n][1], fmaf(ba, qSum[G][n][1], s[sub][n][1]));
                        s[sub][n][2] = fmaf(sb, acc[n][2], fmaf(bb, qSum[G][n][0], s[sub][n][2]));
                        s[sub][n][3] = fmaf(sb, acc[n][3], fmaf(bb, qSum[G][n][1], s[sub][n][3]));
                    }
                }
            }
            if (careful || (broken[0] | broken[1])) {
                // a row r of a subtile is the first or second key of pair r / 2
                const uint32_t marks0 = broken[0] | (broken[0] >> 16), marks1 = broken[1] | (broken[1] >> 16);
#pragma unroll
                for (int sub = 0; sub < 2; ++sub)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const bool bad = (g & 1u ? marks1 : marks0) >> (8 * sub + 4 * h + (g >> 1)) & 1u;
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                const uint32_t column = column0 + 8 * n + (2 * t + c) % kColumns;
                                if (!sees(j0 + 16 * sub + 8 * h + (int)keyA, w.q.p0 + (int)(column / group))) s[sub][n][2 * h + c] = -INFINITY;
                                else if (bad) s[sub][n][2 * h + c] = NAN;
                            }
                    }
            }

            // ---- weights ----
            bool above = false;
            float most[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float m = fmaxf(fmaxf(s[0][n][c], s[0][n][c + 2]), fmaxf(s[1][n][c], s[1][n][c + 2]));
                    m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 4));
                    m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 8));
                    m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 16));
                    most[n][c] = m * toLog2[n][c];
                    above |= most[n][c] > top[n][c] + kLazy;
                }
            if (__any_sync(0xFFFFFFFFu, above)) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float f[2];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float next = fmaxf(top[n][c], most[n][c]);
                        f[c] = exp2_fast(top[n][c] - next);
                        top[n][c] = next;
                    }
#pragma unroll
                    for (int G = 0; G < NG; ++G)
#pragma unroll
                        for (int v = 0; v < 4; ++v)
#pragma unroll
                            for (int k = 0; k < 4; ++k) o[G][v][n][k] *= f[k & 1];
#pragma unroll
                    for (int k = 0; k < 4; ++k) extra[n][k] *= f[k & 1];
                }
            }
            uint32_t p[2][NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int sub = 0; sub < 2; ++sub)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        p[sub][n][h] = transposed(pack_f16(exp2_fast(fmaf(s[sub][n][2 * h], toLog2[n][0], -top[n][0])), exp2_fast(fmaf(s[sub][n][2 * h + 1], toLog2[n][1], -top[n][1]))));
            }

            // ---- values; row 8 of the last product adds up the weights, rows 0 .. NG - 1 the biases ----
            const uint32_t ones = g == 0 ? 0x3C003C00u : 0u;
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                uint32_t bias[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t from = (NG == 1 ? 0u : (g & 1u) * 16) + 8 * sub + 4 * h + t;
                    bias[h] = __shfl_sync(0xFFFFFFFFu, pairBias[0], from);
                    if (NG == 4) {
                        const uint32_t other = __shfl_sync(0xFFFFFFFFu, pairBias[kPairs - 1], from);
                        if (g & 2u) bias[h] = other;
                    }
                    if (g >= (uint32_t)NG) bias[h] = 0u;
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) mma_f16(extra[n], bias[0], ones, bias[1], ones, p[sub][n][0], p[sub][n][1]);
                const uint32_t row = base + subRow[sub] * CB;
#pragma unroll
                for (int G = 0; G < NG; ++G) {
                    uint32_t lo[2], hi[2], scale[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t wa = lds32(row + vOff[0][G] + 8 * h * CB), wb = lds32(row + vOff[1][G] + 8 * h * CB);
                        lo[h] = __byte_perm(wa, wb, 0x5410);
                        hi[h] = __byte_perm(wa, wb, 0x7632);
                        scale[h] = __shfl_sync(0xFFFFFFFFu, pairScale[NG == 4 ? G / 2 : 0], (G & 1) * 16 + 8 * sub + 4 * h + t);
                    }
                    const uint32_t lo0 = lo[0] >> 8, lo1 = lo[1] >> 8, hi0 = hi[0] >> 8, hi1 = hi[1] >> 8;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        uint32_t b0 = mul_f16x2(p[sub][n][0], scale[0]), b1 = mul_f16x2(p[sub][n][1], scale[1]);
                        const uint32_t rest0 = residual_f16x2(p[sub][n][0], scale[0], b0), rest1 = residual_f16x2(p[sub][n][1], scale[1], b1);
                        if (SPLIT && g >= 4) b0 = rest0, b1 = rest1;
                        mma_f16(o[G][0][n], nibbles<0>(lo[0], lo0), nibbles<0>(hi[0], hi0), nibbles<0>(lo[1], lo1), nibbles<0>(hi[1], hi1), b0, b1);
                        mma_f16(o[G][1][n], nibbles<1>(lo[0], lo0), nibbles<1>(hi[0], hi0), nibbles<1>(lo[1], lo1), nibbles<1>(hi[1], hi1), b0, b1);
                        mma_f16(o[G][2][n], nibbles<2>(lo[0], lo0), nibbles<2>(hi[0], hi0), nibbles<2>(lo[1], lo1), nibbles<2>(hi[1], hi1), b0, b1);
                        mma_f16(o[G][3][n], nibbles<3>(lo[0], lo0), nibbles<3>(hi[0], hi0), nibbles<3>(lo[1], lo1), nibbles<3>(hi[1], hi1), b0, b1);
                        if (!SPLIT) {
                            mma_f16(o[G][0][n], nibbles<0>(lo[0], lo0), nibbles<0>(hi[0], hi0), nibbles<0>(lo[1], lo1), nibbles<0>(hi[1], hi1), rest0, rest1);
                            mma_f16(o[G][1][n], nibbles<1>(lo[0], lo0), nibbles<1>(hi[0], hi0), nibbles<1>(lo[1], lo1), nibbles<1>(hi[1], hi1), rest0, rest1);
                            mma_f16(o[G][2][n], nibbles<2>(lo[0], lo0), nibbles<2>(hi[0], hi0), nibbles<2>(lo[1], lo1), nibbles<2>(hi[1], hi1), rest0, rest1);
                            mma_f16(o[G][3][n], nibbles<3>(lo[0], lo0), nibbles<3>(hi[0], hi0), nibbles<3>(lo[1], lo1), nibbles<3>(hi[1], hi1), rest0, rest1);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(barEmpty + 8 * stage);
        }

        // ---- the warps' outputs joined ----
        const float unscale = power_of_two(E);
        const bool mineToo = !SPLIT || t < 2;  // columns 4 .. 7 are the rests of columns 0 .. 3
        if (SPLIT)
#pragma unroll
            for (int G = 0; G < NG; ++G)
#pragma unroll
                for (int v = 0; v < 4; ++v)
#pragma unroll
                    for (int k = 0; k < 4; ++k) o[G][v][0][k] += __shfl_xor_sync(0xFFFFFFFFu, o[G][v][0][k], 2);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                if (!mineToo) continue;
                if (g == 0) joinStats[warp][8 * n + 2 * t + c] = make_float2(top[n][c], extra[n][2 + c]);
                if (g < (uint32_t)NG) joinBias[warp][g][8 * n + 2 * t + c] = extra[n][c] * unscale;
            }
        named_barrier(1, 32 * kConsumers);
        float *mine = joined + (warp & 1u) * kColumns * (DIM + 4);
#pragma unroll
        for (int turn = 0; turn < 2; ++turn) {
            if ((int)(warp >> 1) == turn && mineToo) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const uint32_t column = 8 * n + 2 * t + c;
                        float all = joinStats[0][column].x;
#pragma unroll
                        for (int k = 1; k < kConsumers; ++k) all = fmaxf(all, joinStats[k][column].x);
                        const float f = exp2_fast(top[n][c] - all);
#pragma unroll
                        for (int G = 0; G < NG; ++G) {
                            const float bias = joinBias[warp][G][column];
#pragma unroll
                            for (int v = 0; v < 4; ++v)
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    float *to = mine + column * (DIM + 4) + 64 * G + 8 * g + v + 4 * h;
                                    // (a weight of zero times an output that is none is none: a warp that saw a NaN has a NaN sum)
                                    const float value = f * fmaf(o[G][v][n][2 * h + c] * (v % 2 ? 0x1p20f : 0x1p24f), unscale, bias);
                                    *to = turn ? *to + value : value;
                                }
                        }
                    }
            }
            named_barrier(1, 32 * kConsumers);
        }

        // ---- the unit's rows, or this CTA's part of them ----
        const uint32_t used = min(kColumns, columns - column0);
        const bool whole = count == unitTiles;
        const uint32_t slot = 2 * cta + (t0 == 0 ? 1u : 0u);
        auto write = [&](uint32_t column, uint32_t at, const float4 &v, float weights) {
            const float f = weights == 0.0f ? 0.0f : 1.0f / weights;
            const uint32_t global = column0 + column;
            uint16_t *to = a.out + (size_t)(w.q.firstRow + global / group) * a.outStride + (head * group + global % group) * DIM + at;
            *reinterpret_cast<uint2 *>(to) = make_uint2(pack_bf16x2(v.x * f, v.y * f), pack_bf16x2(v.z * f, v.w * f));
        };
        for (uint32_t e = tid; e < used * (DIM / 4); e += 32 * kConsumers) {
            const uint32_t column = e / (DIM / 4), at = e % (DIM / 4) * 4;
            const float4 u = *reinterpret_cast<const float4 *>(joined + column * (DIM + 4) + at);
            const float4 v = *reinterpret_cast<const float4 *>(joined + (kColumns + column) * (DIM + 4) + at);
            float all = joinStats[0][column].x, weights = 0.0f;
#pragma unroll
            for (int k = 1; k < kConsumers; ++k) all = fmaxf(all, joinStats[k][column].x);
#pragma unroll
            for (int k = 0; k < kConsumers; ++k) weights += joinStats[k][column].y * exp2_fast(joinStats[k][column].x - all);
            const float4 sum4 = make_float4(u.x + v.x, u.y + v.y, u.z + v.z, u.w + v.w);
            if (whole) {
                write(column, at, sum4, weights);
            } else {
                *reinterpret_cast<float4 *>(args.partials + ((size_t)slot * kColumns + column) * DIM + at) = sum4;
                if (at == 0) args.stats[slot * kColumns + column] = make_float2(all, weights);
            }
        }
        if (!whole) {
            const uint32_t c0 = cta_of(w.first + kUnitCost), c1 = cta_of(w.first + kUnitCost + unitTiles - 1), parts = c1 - c0 + 1;
            // whether this is the last of `expected` CTAs; then what they wrote is there
            auto arrive = [&](uint32_t *counter, uint32_t expected) {
                named_barrier(1, 32 * kConsumers);
                if (tid == 0) {
                    __threadfence();  // (cumulative: for the parts that the barrier made this thread see)
                    const uint32_t n = atomicAdd(counter, 1u);
                    __threadfence();
                    lastPart = n == expected - 1;
                    if (n == expected - 1) *counter = 0u;
                }
                named_barrier(1, 32 * kConsumers);
                return lastPart != 0u;
            };
            // parts of CTAs from, from + step, ... joined, into the unit's rows or the first one's place
            auto join = [&](uint32_t from, uint32_t count, uint32_t step, bool last) {
                auto slot_of = [&](uint32_t c) { return 2 * c + (c == c0 ? 1u : 0u); };
                for (uint32_t e = tid; e < used * (DIM / 4); e += 32 * kConsumers) {
                    const uint32_t column = e / (DIM / 4), at = e % (DIM / 4) * 4;
                    // kAtOnce parts' loads in flight: one after the other they took 10 us for 37 parts
                    constexpr uint32_t kAtOnce = 10;
                    float all = kNone, weights = 0.0f;
                    float4 sum4 = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (uint32_t k0 = 0; k0 < count; k0 += kAtOnce) {
                        float2 st[kAtOnce];
                        float4 v[kAtOnce];
#pragma unroll
                        for (uint32_t k = 0; k < kAtOnce; ++k) {
                            st[k] = make_float2(kNone, 0.0f);
                            v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            if (k0 + k < count) {
                                const uint32_t slot = slot_of(from + (k0 + k) * step);
                                st[k] = __ldcg(args.stats + slot * kColumns + column);
                                v[k] = __ldcg(reinterpret_cast<const float4 *>(args.partials + ((size_t)slot * kColumns + column) * DIM + at));
                            }
                        }
                        float next = all;
#pragma unroll
                        for (uint32_t k = 0; k < kAtOnce; ++k) next = fmaxf(next, st[k].x);
                        const float keep = exp2_fast(all - next);
                        all = next;
                        weights *= keep;
                        sum4.x *= keep, sum4.y *= keep, sum4.z *= keep, sum4.w *= keep;
#pragma unroll
                        for (uint32_t k = 0; k < kAtOnce; ++k) {
                            const float f = exp2_fast(st[k].x - all);
                            weights = fmaf(st[k].y, f, weights);
                            sum4.x = fmaf(v[k].x, f, sum4.x), sum4.y = fmaf(v[k].y, f, sum4.y), sum4.z = fmaf(v[k].z, f, sum4.z), sum4.w = fmaf(v[k].w, f, sum4.w);
                        }
                    }
                    if (last) {
                        write(column, at, sum4, weights);
                    } else {
                        *reinterpret_cast<float4 *>(args.partials + ((size_t)slot_of(from) * kColumns + column) * DIM + at) = sum4;
                        if (at == 0) joinStats[0][column] = make_float2(all, weights);
                    }
                }
                if (!last) {
                    named_barrier(1, 32 * kConsumers);  // (the first one's maxima have been read)
                    if (tid < used) args.stats[slot_of(from) * kColumns + tid] = joinStats[0][tid];
                }
            };
            // by groups of 16 first where there are more: one CTA would take 100 us for 296 parts (a CTA is the first of one unit
            // and inside another at most: a group's counter goes by which)
            constexpr uint32_t kGroupParts = 16;
            const uint32_t groups = (parts + kGroupParts - 1) / kGroupParts, group0 = c0 + (cta - c0) / kGroupParts * kGroupParts;
            bool last = groups == 1;
            uint32_t *counter = args.arrived + (last ? 0 : group0 == c0 ? 1 : 2) * gridDim.x + group0;
            uint32_t from = group0, many = min(kGroupParts, c1 - group0 + 1), step = 1;
#pragma unroll 1
            while (arrive(counter, many)) {
                join(from, many, step, last);
                if (last) break;
                last = true;
                counter = args.arrived + c0;
                from = c0, many = groups, step = kGroupParts;
            }
        }
        n0 += count;
        named_barrier(1, 32 * kConsumers);  // the joining buffers are free
    } while (next_unit(w));
    if (lane == 0 && abortFlag) *a.errorFlag = kFlagWait;
}

KernelSmemMemo rowsMemo[3][3];

template <int DIM, int NT, bool SPLIT = false>
bool launch_rows(FFAttention *att, KernelSmemMemo &memo, const CUtensorMap &codes, const CUtensorMap &words, const RowsArgs &args, cudaStream_t stream, const char **error) {
    const size_t smem = rows_smem(DIM, NT);
    int perSm = 0;
    if (!memo.prepare(k_attend_rows<DIM, NT, SPLIT>, att->device, smem, kRowsThreads, &perSm, error)) return false;
    const uint32_t grid = std::min((uint32_t)(att->smCount * std::max(1, perSm)), att->rowsCtas);
    return launched(att, launch_pdl(k_attend_rows<DIM, NT, SPLIT>, dim3(grid), dim3(kRowsThreads), smem, stream, codes, words, args), "k_attend_rows", error);
}

}  // namespace

bool make_pages_maps(CUtensorMap *codes, CUtensorMap *words, const AttendArgs &a, uint32_t dim, uint32_t sides, const char **error) {
    const EncodeTiledFn encode = encode_tiled(error);
    if (!encode) return false;
    const cuuint32_t piece = std::min(kTileKeys, a.page.pageTokens), groups = dim / kGroup, elem[4] = {1, 1, 1, 1};
    const cuuint64_t blocks = (cuuint64_t)a.pageCount * a.kvHeads;
    const cuuint64_t dims[4] = {dim / 2, a.page.pageTokens, 2, blocks}, strides[3] = {dim / 2, a.page.values, a.page.blockBytes};
    const cuuint32_t box[4] = {dim / 2, piece, sides, 1};
    CUresult rc = encode(codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<uint8_t *>(a.pages), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         dim == 256 ? CU_TENSOR_MAP_SWIZZLE_128B : dim == 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc == CUDA_SUCCESS) {
        const cuuint64_t wordDims[3] = {a.page.pageTokens * groups, 2, blocks}, wordStrides[2] = {a.page.values, a.page.blockBytes};
        const cuuint32_t wordBox[3] = {piece * groups, 2, 1};
        rc = encode(words, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<uint8_t *>(a.pages) + a.page.keyWords, wordDims, wordStrides, wordBox, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    }
    if (rc != CUDA_SUCCESS) return fail(error, "cuTensorMapEncodeTiled(cache pages) failed: " + std::to_string((int)rc));
    return true;
}

uint32_t attend_rows_ctas(int smCount) { return 2u * (uint32_t)smCount; }

bool launch_attend_rows(FFAttention *att, const AttendArgs &a, cudaStream_t stream, const char **error) {
    const uint32_t dim = att->cfg.headDim;
    RowsArgs args{a, att->partials, reinterpret_cast<float2 *>(att->stats), att->arrived, (uint32_t)__builtin_ctz(att->cfg.pageTokens), (uint32_t)__builtin_ctz(std::min(kTileKeys, a.page.pageTokens))};
    CUtensorMap codes, words;
    if (!make_pages_maps(&codes, &words, a, dim, 2, error)) return false;
    const uint32_t columns = a.maxRows * (a.heads / a.kvHeads);
    if (dim == 256) {
        if (columns <= 4) return launch_rows<256, 1, true>(att, rowsMemo[0][0], codes, words, args, stream, error);
        if (columns <= 8) return launch_rows<256, 1>(att, rowsMemo[0][1], codes, words, args, stream, error);
        return launch_rows<256, 2>(att, rowsMemo[0][2], codes, words, args, stream, error);
    }
    if (dim == 128) {
        if (columns <= 4) return launch_rows<128, 1, true>(att, rowsMemo[1][0], codes, words, args, stream, error);
        if (columns <= 8) return launch_rows<128, 1>(att, rowsMemo[1][1], codes, words, args, stream, error);
        return launch_rows<128, 2>(att, rowsMemo[1][2], codes, words, args, stream, error);
    }
    if (columns <= 4) return launch_rows<64, 1, true>(att, rowsMemo[2][0], codes, words, args, stream, error);
    if (columns <= 8) return launch_rows<64, 1>(att, rowsMemo[2][1], codes, words, args, stream, error);
    return launch_rows<64, 2>(att, rowsMemo[2][2], codes, words, args, stream, error);
}

}  // namespace ff

// Attention of more than 16 columns a key/value head (verify blocks, prefill chunks) over the paged INT4 cache, on tcgen05.
//
// A row tile is up to 128 rows of one request and key/value head (tokens times the query heads that share the head).
// A unit of work is one row tile; its keys are tiles of 64, and all units' tiles end to end are cut into equal runs, one
// per CTA, one CTA per SM.  A unit that several CTAs share is joined by whichever of them ends last, in the CTAs' order.
//
// Per key tile, warp by role: two copy packed codes, keys' with the scale words and values'; one turns the tile's scale words into the pairs that
// the expansion multiplies with; sixteen expand codes to f16 tiles in shared memory (128-byte swizzle, keys and values alike
// [64 values][key][128 bytes]), four a slot, so that one group's waits stand behind the other's arithmetic; one issues the MMAs; two
// warpgroups own a row a thread and take the tiles in turn:
//   S = Q K^T   A: the rows' queries, in tensor memory for the whole unit (from shared memory an MMA of 64 keys takes 73
//               cycles, from tensor memory 33); B: the keys, K-major
//   P = 2^(S f + E - M)   in registers, back into S's columns as f16; their sum at the largest logit, without E
//   O += P V    A: P; B: the values, N-major; O stays in tensor memory
// A tile's warpgroup waits for the maximum M that the one before it settled on, not for its weights; M moves, and O with it, only
// where a row passes it by 2^8.  (Both warpgroups on each tile, half a row a thread, were slower: what a tile costs besides its
// arithmetic was paid twice.)
// Tensor memory: Q dim/2, O dim, S tiles of 64 columns, two at dim 256 (512 in all, which is all there is), four below.
//
// f16 holds 11 bits of keys, values and weights where bf16 would hold 8; its range is kept by powers of two: a row's
// own for the queries, a tile's own for keys (taken back with the logits) and for values (E, part of the exponent of P and
// of the maximum M that P stays below 2^14 of; keys and values of 2^116 and more are out of its reach).  Lost is what of a key or value is
// below 2^-20 of the largest of its tile, and a weight whose product with its tile's largest value is below 2^-30 of the largest such of its
// part of the keys; it is in the sum of the weights all the same, which does not know E.  A code masked in place is the f16 code * 2^-24 or * 2^-20, and one FMA with scale times 2^24 or
// 2^20 and the bias rounds once: nine instructions a word of eight codes.
//
// 4096 rows of 16 heads of 256 over 36864 keys take 2.2 ms, 1.06 PFLOP/s: 63 % of the burst bf16 rate, 75 % of the sustained one
// (at 36864 keys the power limit holds the clock below its maximum).  A tile takes 1.0 to 1.2 us.  Its MMAs alone are 1077 cycles: 16 of
// 32.8 and 4 of 138, each form timed by itself.  The tensor pipe is active 45 % of the time at 8192 keys: S of a tile waits in one of
// two buffers until its weights are formed, and tensor memory has no third at 256 values a head.  4096 rows in a window of 1024 take
// 133 us: 19 tiles a unit, beside which queries, first logits, output and parts of units count; five ragged requests of up to
// 613 rows with 14 heads of 64 28 us.
//
// Attention behind a shared prefix is three launches: this kernel with the groups' rows over their prefixes, whose units' parts stay apart; a join;
// then the requests' rows from behind the prefixes, here or in the kernel for few rows, what the join gave added to their own.  64 requests with
// 256 columns a key/value head behind 32768 keys of 8 heads of 128 take 83 us with up to 2048 keys of their own: 1.27 us for 1024 keys of the prefix (0.73 a tile of 128 columns
// and CTA), 14 more than with 64 keys of their own, the rest whatever the lengths.  The requests' launch begins while the join runs.  Read by request they take 565.  With fewer columns or keys the
// launches cost more than they save (ff_attention.cu).  In copies that skip a part (for the time alone) a tile takes at 64, 128 and 256 values a head 0.57,
// 0.74 and 1.0 us, without the expansion 0.55, 0.66 and 0.77, without exponentials 0.58, 0.72 and 0.96, with a quarter of the products 0.59, 0.74 and
// 0.92: up to 128 values a chain of hand-overs, not one unit, sets the pace.  A second warp for the scales (32 warps, 40 registers) was slower: 0.61, 0.78.
#include <algorithm>
#include <string>

#include "ff_attention_device.cuh"

namespace ff {

namespace {

// warps by role: copies of keys, MMAs, scales, copies of values; expansion; rows
constexpr int kKeyCopyWarp = 0, kMmaWarp = 1, kScaleWarp = 2, kValueCopyWarp = 3, kDequantWarps = 16, kRowGroups = 2;
constexpr int kFirstDequant = 4, kFirstRowWarp = kFirstDequant + kDequantWarps, kRowWarps = 4 * kRowGroups;
constexpr int kTilesThreads = 32 * (kFirstRowWarp + kRowWarps);
// registers a thread by role: together no more than the launch's 72 each (4096 rows over 36864 keys, one after the other on one
// card: eight expanding warps 2.34 ms, twelve 2.12 to 2.14, sixteen 2.01)
constexpr int kRegsOthers = 48, kRegsRows = 128;
static_assert(128 * kRegsOthers + 32 * kDequantWarps * kRegsOthers + 32 * kRowWarps * kRegsRows <= kTilesThreads * 72, "register split");
constexpr uint32_t kRows = kTileRows;
// Weights are held times 2^6 (as is their sum): with the 2^8 that a logit may pass the maximum by they stay within f16, and what
// is 2^-30 of the largest is still something.
constexpr float kWeightScale = 6.0f;
constexpr uint32_t kUnitCost = 8;  // tiles' time that a unit takes besides its tiles
constexpr uint32_t kSlots = 4;  // expanded tiles
__host__ __device__ constexpr uint32_t packed_tiles(int dim) { return dim == 128 ? 4u : 3u; }  // packed ones, of keys and of values each
// S has as many buffers as tensor memory has room for beside queries and outputs; its products run as far ahead of those of the weights as
// the rings allow; scales and exponents are kept for that many tiles and as many more.  us a tile and CTA (full row tiles, three and four tiles
// ahead): 64 values a head 0.57 with three, 0.60 with four; 128 0.75 with three, 0.72 with four.
__host__ __device__ constexpr uint32_t score_buffers(int dim) { return dim == 256 ? 2u : 4u; }
__host__ __device__ constexpr uint32_t tiles_ahead(int dim) { return dim == 256 ? 2u : dim == 128 ? 4u : 3u; }
__host__ __device__ constexpr uint32_t info_tiles(int dim) { return dim == 256 ? 4u : 8u; }
// The expansion's items are the keys of as many tiles, then values and keys in turn, at the end of a unit the values that are left: no more
// values than that one behind the other.  So the values packed_tiles before a tile's are at least one item more before.
// A wait for O of a tile is by parity: the tile score_buffers before, whose product counts on the same barrier, is done when the tile's S is (S runs
// no further ahead).
__host__ __device__ constexpr bool rings_hold(int dim) { return packed_tiles(dim) + 1 >= kSlots && tiles_ahead(dim) <= packed_tiles(dim) && tiles_ahead(dim) <= score_buffers(dim); }
static_assert(rings_hold(64) && rings_hold(128) && rings_hold(256), "a free slot says that the ring's place was read; a buffer each");

struct TilesArgs {
    AttendArgs a;
    float *partials;      // [2 CTAs][rows][DIM]
    float4 *stats;        // [2 CTAs][rows] M, the largest logit L, the weights' sum at 2^L
    uint32_t *arrived;    // [3][CTAs], zero between launches: of a unit, of its first group of parts, of another group
    uint32_t pageShift, pieceShift, tileTokens;  // log2 of a page's tokens and of the keys of a tile on one page; tokens of a row tile
};

__host__ __device__ constexpr uint32_t slot_bytes(int dim) { return kTileKeys * dim * 2; }
__host__ __device__ constexpr uint32_t packed_bytes(int dim) { return (kTileKeys * dim / 2 + 1023u) & ~1023u; }
__host__ __device__ constexpr uint32_t words_bytes(int dim) { return 2u * kTileKeys * (dim / 64) * 4u; }  // of a tile, keys' and values'
__host__ __device__ constexpr uint32_t tiles_smem(int dim) { return 1024u + kSlots * slot_bytes(dim) + 2 * packed_tiles(dim) * packed_bytes(dim) + (info_tiles(dim) + packed_tiles(dim)) * words_bytes(dim); }

// K-major or N-major tile of f16 with the 128-byte swizzle: rows of 128 bytes, groups of eight 1024 bytes apart; N-major:
// the next 64 values `lead` bytes further.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr, uint32_t lead) {
    uint64_t d = (uint64_t)((addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(lead >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
// f16 x f16 -> fp32, 128 rows, n columns
__device__ __forceinline__ uint32_t idesc_f16(uint32_t n, bool bNMajor) { return (1u << 4) | ((bNMajor ? 1u : 0u) << 16) | ((n >> 3) << 17) | ((128u >> 4) << 24); }
__device__ __forceinline__ void mma_a_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
        "}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
constexpr uint32_t kWaitLimit = 1u << 20;
// The bounded waits of ff_tc_device.cuh without a call: a kernel that divides its registers among the roles has none.
template <bool kSleep>
__device__ __forceinline__ bool wait_lane(uint32_t bar, uint32_t parity, volatile uint32_t *abortFlag) {
    if (mbar_try_wait(bar, parity)) return true;
#pragma unroll 1
    for (uint32_t i = 0; i < kWaitLimit; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if (kSleep) __nanosleep(40);
        if ((i & 255u) == 255u && *abortFlag) return false;
    }
    *abortFlag = 1u;
    return false;
}
template <bool kSleep>
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile uint32_t *abortFlag) {
    return __all_sync(0xFFFFFFFFu, wait_lane<kSleep>(bar, parity, abortFlag));
}
// The last wait of a role for what it issued, also after another one gave up.
__device__ __forceinline__ void landed(uint32_t bar, uint32_t parity) {
#pragma unroll 1
    for (uint32_t i = 0; i < kWaitLimit && !mbar_try_wait(bar, parity); ++i) __nanosleep(40);
    __syncwarp();
}
// two fp32 operations an instruction
__device__ __forceinline__ unsigned long long pair_f32(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float first_f32(unsigned long long v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float second_f32(unsigned long long v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ unsigned long long fma_f32x2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ unsigned long long add_f32x2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}

// the n lowest bits of 64
__device__ __forceinline__ unsigned long long first_bits(long long n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull; }
// bit l to bit 2 l
__device__ __forceinline__ unsigned long long spread_bits(uint32_t v) {
    unsigned long long x = v;
    x = (x | x << 16) & 0x0000FFFF0000FFFFull;
    x = (x | x << 8) & 0x00FF00FF00FF00FFull;
    x = (x | x << 4) & 0x0F0F0F0F0F0F0F0Full;
    x = (x | x << 2) & 0x3333333333333333ull;
    return (x | x << 1) & 0x5555555555555555ull;
}

// What a launch's "requests" are.  Prefix: the groups of requests that share a prefix, whose rows all see its keys; results go to
// args.a.shared, not yet out.  Suffix: requests from behind their group's prefix on, what the prefix gave joined to it.
enum class TilesOf { kRequest, kPrefix, kSuffix };

// A row tile of a request as the kernel sees it.
struct RowTileOf {
    uint32_t r, firstRow, tokens;          // its request, first row of q, tokens
    int p0;                                // position of its first token
    uint32_t tilesSink, lowTile, tiles;    // key tiles: the first tilesSink, then from lowTile on
};
struct SharedTileOf : RowTileOf {
    bool joins;  // suffix: whether the rows have a prefix
};

template <int DIM, TilesOf OF>
__global__ void __launch_bounds__(kTilesThreads, 1) k_attend_tiles(const __grid_constant__ CUtensorMap mapCodes, const __grid_constant__ CUtensorMap mapWords, const TilesArgs args) {
    constexpr bool kPrefix = OF == TilesOf::kPrefix, kSuffix = OF == TilesOf::kSuffix;
    using RowTile = std::conditional_t<OF == TilesOf::kRequest, RowTileOf, SharedTileOf>;
    using Known = std::conditional_t<OF == TilesOf::kRequest, uint3, uint4>;  // first row, rows, length; prefix: its request; suffix: its prefix's keys
    constexpr int NG = DIM / 64, CB = DIM / 2, WB = NG * 4;
    constexpr uint32_t kSlot = slot_bytes(DIM), kPack = packed_bytes(DIM);
    constexpr uint32_t kWordSide = words_bytes(DIM) / 2, kUnits = kTileKeys * NG;  // of a slot: a key's group of 64 values
    // (no more groups than slots: one that waited for a slot two rounds ahead would take one round's parity for the other's)
    constexpr uint32_t kGroupWarps = DIM == 64 ? 2 : 4, kGroups = kDequantWarps / kGroupWarps < kSlots ? kDequantWarps / kGroupWarps : kSlots, kUnitsEach = kUnits / (32 * kGroupWarps);
    constexpr uint32_t kPacked = packed_tiles(DIM), kInfo = info_tiles(DIM), kBuffers = score_buffers(DIM), kAhead = tiles_ahead(DIM);
    constexpr uint32_t kColQ = 0, kColO = DIM / 2, kColS = kColO + DIM;
    extern __shared__ uint8_t tilesSmem[];
    __shared__ __align__(8) uint64_t barriers[2 * kSlots + 4 * kPacked + 2 * kInfo + 4 * kBuffers + 1 + 1 + 8 + 1];
    __shared__ uint32_t tmemSlot, lastPart;
    __shared__ volatile uint32_t abortFlag;
    __shared__ uint32_t firstTile[kTilesThreads + 1], firstWork[kTilesThreads + 1], warpSums[32];
    __shared__ uint32_t holes[kPacked], hidden[kInfo][2];
    __shared__ float4 tileInfo[kInfo];
    __shared__ Known known[kTilesThreads];
    __shared__ float topShared[kRows], sumShared[kRowGroups][kRows], refShared[kRowGroups][kRows];
    __shared__ uint32_t largestShared[kRowGroups][kRows];
    const AttendArgs &a = args.a;
    const uint32_t tid = threadIdx.x, warp = (uint32_t)warp_index(), lane = tid & 31u;
    const uint32_t slots = (sm_addr(tilesSmem) + 1023u) & ~1023u, packed = slots + kSlots * kSlot, scales = packed + 2 * kPacked * kPack, words = scales + kInfo * words_bytes(DIM);
    const uint32_t group = a.heads / a.kvHeads;
    const uint32_t bar0 = sm_addr(barriers);
    const uint32_t barTile = bar0, barTileFree = barTile + 8 * kSlots, barPack = barTileFree + 8 * kSlots, barPackFree = barPack + 16 * kPacked;  // keys', then values'
    const uint32_t barInfo = barPackFree + 16 * kPacked, barInfoFree = barInfo + 8 * kInfo;
    const uint32_t barS = barInfoFree + 8 * kInfo, barP = barS + 8 * kBuffers, barO = barP + 16 * kBuffers, barQ = barO + 8 * kBuffers, barJoin = barQ + 8, barTop = barJoin + 8, barDone = barTop + 64;
    if (tid == 0) {
        abortFlag = 0;
        for (uint32_t s = 0; s < kSlots; ++s) {
            mbar_init(barTile + 8 * s, kGroupWarps);
            mbar_init(barTileFree + 8 * s, 1);
        }
        for (uint32_t s = 0; s < 2 * kPacked; ++s) {
            mbar_init(barPack + 8 * s, 1);
            mbar_init(barPackFree + 8 * s, kGroupWarps + (s < kPacked ? 1 : 0));  // (keys: and the scale warp)
        }
        for (uint32_t s = 0; s < kInfo; ++s) {
            mbar_init(barInfo + 8 * s, 1);
            mbar_init(barInfoFree + 8 * s, 1);
        }
        for (uint32_t s = 0; s < kBuffers; ++s) {
            mbar_init(barS + 8 * s, 1);
            mbar_init(barP + 16 * s, 4);  // the first 32 keys' weights
            mbar_init(barP + 16 * s + 8, 4);
            mbar_init(barO + 8 * s, 1);
        }
        mbar_init(barQ, kRowWarps);
        mbar_init(barJoin, kRowWarps);
        for (uint32_t s = 0; s < 8; ++s) mbar_init(barTop + 8 * s, 1);
        mbar_init(barDone, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == (uint32_t)kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sm_addr(&tmemSlot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, tmemSlot, 0);
    // (Behind the launch over the prefixes this one begins while that ends: what it reads of the caller's is from before both.)
    if (!kSuffix) pdl_enter();

    // ---- the plan: row tiles of the requests, key tiles of those, this CTA's run ----
    // A request: its first row, rows, length; looked up once where there is a thread for each.
    const uint32_t requests = kPrefix ? a.shared.groups : a.requests, run = (requests + kTilesThreads - 1) / kTilesThreads;
    auto look_up = [&](uint32_t r) {
        if constexpr (kPrefix) {
            const SharedGroup g = shared_group(a, r);
            return make_uint4(g.firstRow, g.keys ? g.rows : 0u, g.keys, g.request);
        } else {
            const uint32_t begin = min(__ldg(a.rowStart + r), a.tokens), end = min(__ldg(a.rowStart + r + 1), a.tokens);
            const uint32_t rows = end > begin ? end - begin : 0u, length = min(__ldg(a.lengths + r), 0x7FFFFFFFu);
            if constexpr (kSuffix) return make_uint4(begin, rows, length, rows ? shared_keys(a, r, (int)length - (int)rows) : 0u);
            else return make_uint3(begin, rows, length);
        }
    };
    auto request = [&](uint32_t r) { return run == 1 ? known[r] : look_up(r); };
    auto row_tiles_of = [&](uint32_t r) { return (min(request(r).y, a.maxRows) + args.tileTokens - 1) / args.tileTokens; };
    auto row_tile = [&](uint32_t r, uint32_t i) {
        RowTile q;
        const Known of = request(r);
        const uint32_t used = min(of.y, a.maxRows);
        q.r = r;
        q.firstRow = of.x + i * args.tileTokens;
        q.tokens = min(args.tileTokens, used - i * args.tileTokens);
        q.p0 = (int)of.z - (int)of.y + (int)(i * args.tileTokens);
        if constexpr (kPrefix) {
            q.r = of.w;
            q.p0 = (int)of.z - 1;  // (every row sees every key)
            q.lowTile = q.tilesSink = 0;
            q.tiles = of.z / kTileKeys;
            return q;
        }
        const uint32_t last = (uint32_t)max(0, q.p0 + (int)q.tokens), ends = (min(last, a.tableKeys) + kTileKeys - 1) / kTileKeys;
        q.lowTile = q.tilesSink = 0;
        if (a.window) {
            const uint32_t low = (uint32_t)max((long long)0, (long long)q.p0 - (long long)a.window + 1);
            q.lowTile = min(low / kTileKeys, ends);
            q.tilesSink = min((uint32_t)(((unsigned long long)a.sinks + kTileKeys - 1) / kTileKeys), q.lowTile);
        }
        if constexpr (kSuffix) {
            q.joins = of.w != 0u;
            q.lowTile = of.w / kTileKeys;
        }
        q.tiles = max(1u, q.tilesSink + ends - q.lowTile);  // (rows without keys: one tile that nobody sees)
        return q;
    };
    auto block_scan = [&](uint32_t sum, uint32_t *first) {  // first[t]: sum over the threads before t
        uint32_t scan = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, scan, d);
            if (lane >= (uint32_t)d) scan = add_work(scan, v);
        }
        if (lane == 31u) warpSums[warp] = scan;
        __syncthreads();
        const uint32_t mine = lane < kTilesThreads / 32 ? warpSums[lane] : 0u;
        uint32_t sums = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, sums, d);
            if (lane >= (uint32_t)d) sums = add_work(sums, v);
        }
        const uint32_t total = __shfl_sync(0xFFFFFFFFu, sums, 31);
        first[tid] = __shfl_sync(0xFFFFFFFFu, sums - mine, warp) + scan - sum;
        if (tid == 0) first[kTilesThreads] = total;
        __syncthreads();
        return total;
    };
    const uint32_t r0 = min(tid * run, requests), r1 = min(r0 + run, requests);
    // rowStart goes back, to rows that several requests would write: such a call is refused like one with too much work
    auto goes_back = [&](uint32_t r) {
        if constexpr (kPrefix) return false;  // (the requests' launch looks, and then takes nothing from this one)
        else return __ldg(a.rowStart + r + 1) < __ldg(a.rowStart + r);
    };
    uint32_t mineTiles = 0;
    for (uint32_t r = r0; r < r1; ++r) {
        const Known of = look_up(r);
        if (run == 1) known[r] = of;
        mineTiles = goes_back(r) ? kTooMuch : add_work(mineTiles, (min(of.y, a.maxRows) + args.tileTokens - 1) / args.tileTokens);
        if (!kPrefix && of.y && (int)of.z - (int)of.y + (int)min(of.y, a.maxRows) > 0 && of.z - of.y + min(of.y, a.maxRows) > a.tableKeys) *a.errorFlag = kFlagTableRow;  // (what the row has no room for is not walked)
    }
    if (kSuffix && groups_go_back(a, tid, kTilesThreads)) mineTiles = kTooMuch;
    const uint32_t allTiles = block_scan(mineTiles, firstTile);
    const uint32_t rowTiles = allTiles == kTooMuch ? 0u : allTiles;
    // the n-th row tile
    struct Place {
        uint32_t r, i, count;  // request, row tile of it, row tiles that it has
    };
    auto place_of = [&](uint32_t n) {
        uint32_t low = 0, high = (requests + run - 1) / run;  // (threads that have requests)
        while (high - low > 1) {
            const uint32_t mid = (low + high) >> 1;
            if (firstTile[mid] <= n) low = mid;
            else high = mid;
        }
        n -= firstTile[low];
        Place p{low * run, 0u, 0u};
        for (;; ++p.r) {
            p.count = row_tiles_of(p.r);
            if (n < p.count) break;
            n -= p.count;
        }
        p.i = n;
        return p;
    };
    auto advance = [&](Place &p) {
        if (++p.i < p.count) return;
        p.i = 0;
        do {
            ++p.r;
            p.count = row_tiles_of(p.r);
        } while (p.count == 0);
    };
    const uint32_t perThread = (rowTiles + kTilesThreads - 1) / kTilesThreads;
    const uint32_t n0 = min(tid * perThread, rowTiles), n1 = min(n0 + perThread, rowTiles);
    uint32_t work = 0;
    if (n0 < n1) {
        Place p = place_of(n0);
        for (uint32_t n = n0; n < n1; ++n) {
            work = add_work(work, work_of(row_tile(p.r, p.i).tiles + kUnitCost, a.kvHeads));
            if (n + 1 < n1) advance(p);
        }
    }
    const uint32_t allWork = block_scan(work, firstWork);
    const bool refused = allTiles == kTooMuch || allWork == kTooMuch;  // (the places of units are nothing then)
    const uint32_t total = refused ? 0u : allWork;

    // rows that no unit writes: behind the last request's, and past maxRows
    if constexpr (!kPrefix) {
        const uint32_t covered = a.requests && !refused ? min(__ldg(a.rowStart + a.requests), a.tokens) : 0u;
        const uint32_t perRow = a.heads * DIM / 8;
        for (uint32_t row = covered + blockIdx.x; row < a.tokens; row += gridDim.x)
            for (uint32_t i = tid; i < perRow; i += kTilesThreads) *reinterpret_cast<uint4 *>(a.out + (size_t)row * a.outStride + i * 8) = make_uint4(0u, 0u, 0u, 0u);
        if (blockIdx.x == 0) {
            if (tid == 0 && refused) *a.errorFlag = kFlagWork;
            __syncthreads();
            if (kSuffix && groups_go_back(a, tid, kTilesThreads)) *a.errorFlag = kFlagRows;
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
    const uint32_t ctas = min(gridDim.x, max(1u, total / 2u)), cta = blockIdx.x;
    auto start_of = [&](uint32_t c) { return divided((unsigned long long)c * total, ctas); };
    auto cta_of = [&](uint32_t x) { return divided(((unsigned long long)x + 1) * ctas - 1, total); };
    const uint32_t begin = cta < ctas && total ? start_of(cta) : 0u, end = cta < ctas && total ? start_of(cta + 1) : 0u;

    // The run's segments: consecutive key tiles of one unit, whose tile i stands at x = first + kUnitCost + i.  A unit costs its
    // tiles and kUnitCost more: its queries, first logits and output take as long.
    struct Walk {
        Place place;
        RowTile q;
        uint32_t first, head, t0, count;  // segment [t0, t0 + count)
    };
    auto take = [&](Walk &w) {
        const uint32_t tile0 = w.first + kUnitCost;
        w.t0 = begin > tile0 ? min(begin - tile0, w.q.tiles) : 0u;
        w.count = (end > tile0 ? min(end - tile0, w.q.tiles) : 0u) - w.t0;
    };
    auto next_unit = [&](Walk &w) {
        w.first += w.q.tiles + kUnitCost;
        if (w.first >= end) return false;
        if (++w.head == a.kvHeads) {
            w.head = 0;
            advance(w.place);
            w.q = row_tile(w.place.r, w.place.i);
        }
        take(w);
        return true;
    };
    // the segment behind; false past the run's end (a run may begin or end in front of a unit's first tile)
    auto next_segment = [&](Walk &w) {
        do {
            if (!next_unit(w)) return false;
        } while (w.count == 0);
        return true;
    };
    auto first_segment = [&](Walk &w) {
        uint32_t low = 0, high = kTilesThreads;
        while (high - low > 1) {
            const uint32_t mid = (low + high) >> 1;
            if (firstWork[mid] <= begin) low = mid;
            else high = mid;
        }
        w.place = place_of(low * perThread);
        uint32_t n = begin - firstWork[low];
        for (;; advance(w.place)) {
            w.q = row_tile(w.place.r, w.place.i);
            if (n < (w.q.tiles + kUnitCost) * a.kvHeads) break;
            n -= (w.q.tiles + kUnitCost) * a.kvHeads;
        }
        w.head = n / (w.q.tiles + kUnitCost);
        w.first = begin - n % (w.q.tiles + kUnitCost);
        take(w);
        return w.count != 0 || next_segment(w);
    };
    // (by one warp for all: by each for itself it took 5000 cycles, most of them waiting for issue slots)
    __shared__ Walk firstWalk;
    __shared__ bool firstMore;
    if (warp == 0 && begin < end) {
        Walk w;
        const bool more = first_segment(w);
        if (lane == 0) firstWalk = w, firstMore = more;
    }
    __syncthreads();
    auto key_at = [&](const RowTile &q, uint32_t t) { return (t < q.tilesSink ? t : q.lowTile + t - q.tilesSink) * kTileKeys; };
    const uint32_t pieceKeys = 1u << args.pieceShift, pieces = kTileKeys >> args.pieceShift;

    if (warp < (uint32_t)kFirstRowWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOthers));
        if (begin >= end) {
            // nothing
        } else if (warp == (uint32_t)kKeyCopyWarp || warp == (uint32_t)kValueCopyWarp) {
            // ---------------- copies ----------------
            // The warp runs as one and an elected lane issues (a copy in a branch that lanes take apart costs several hundred
            // cycles: its operands go to the uniform registers by a loop over the lanes); without a division in the loop, and keys
            // and values by a warp each: with one for both its chain of latencies, 2300 cycles a tile, was the kernel's pace.
            const uint32_t side = warp == (uint32_t)kKeyCopyWarp ? 0u : 1u;
            const uint32_t full = barPack + 8 * kPacked * side, empty = barPackFree + 8 * kPacked * side, codes = packed + side * kPacked * kPack;
            const uint32_t pieceCodes = CB << args.pieceShift, pieceWords = WB << args.pieceShift, pieceBytes = pieceCodes + (side ? 0u : 2u * pieceWords);
            const uint32_t perTileShift = 6u - args.pieceShift, tilesPer = 32u >> perTileShift;  // pieces of a tile, as a shift; tiles whose pages a warp holds
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            Walk w = firstWalk;
            for (bool more = firstMore; more && ok; more = ok && next_segment(w)) {
                const int keysEnd = w.q.p0 + (int)w.q.tokens;
                // a lane holds the page of one piece of `tilesPer` tiles from `base` on
                auto page_of = [&](uint32_t base) {
                    const uint32_t t = base + (lane >> perTileShift);
                    uint32_t page = FF_NO_PAGE;
                    if (t < w.t0 + w.count) {
                        const uint32_t key = key_at(w.q, t) + ((lane & (pieces - 1u)) << args.pieceShift);
                        if ((int)key < keysEnd) {
                            const uint32_t index = key >> args.pageShift;
                            if (index < a.tableStride) {
                                page = __ldg(a.blockTable + (size_t)w.q.r * a.tableStride + index);
                                if (page >= a.pageCount) *a.errorFlag = kFlagPage;
                            } else {
                                *a.errorFlag = kFlagTableRow;
                            }
                        }
                    }
                    return page;
                };
                const uint32_t tEnd = w.t0 + w.count;
                uint32_t pagesNext = page_of(w.t0);
                for (uint32_t base = w.t0; base < tEnd && ok; base += tilesPer) {
                    const uint32_t pagesNow = pagesNext, many = min(tilesPer, tEnd - base);
                    pagesNext = page_of(base + tilesPer);
                    for (uint32_t i = 0; i < many; ++i) {
                        const uint32_t mine = __shfl_sync(0xFFFFFFFFu, pagesNow, (i << perTileShift) + (lane & (pieces - 1u)));
                        const uint32_t lives = __ballot_sync(0xFFFFFFFFu, lane < pieces && mine < a.pageCount);
                        if (!(ok = wait_warp<true>(empty + 8 * stage, phase ^ 1u, &abortFlag))) break;
                        const uint32_t bar = full + 8 * stage, inTile = key_at(w.q, base + i) & (a.page.pageTokens - 1u);
                        const uint32_t toCodes = codes + stage * kPack, toWords = words + stage * words_bytes(DIM);
                        if (elect_one()) {
                            if (!side) holes[stage] = ~lives;
                            mbar_expect_tx(bar, (uint32_t)__popc(lives) * pieceBytes);
                        }
                        for (uint32_t p = 0; p < pieces; ++p) {
                            const uint32_t block = __shfl_sync(0xFFFFFFFFu, mine, p) * a.kvHeads + w.head, at = (inTile + (p << args.pieceShift)) & (a.page.pageTokens - 1u);
                            if ((lives >> p & 1u) && elect_one()) {
                                tma_load_4d(toCodes + p * pieceCodes, &mapCodes, 0, (int)at, (int)side, (int)block, bar);
                                if (!side) tma_load_3d(toWords + p * 2u * pieceWords, &mapWords, (int)(at * NG), 0, (int)block, bar);
                            }
                        }
                        if (++stage == kPacked) stage = 0, phase ^= 1u;
                    }
                }
            }
            // whatever the other roles did: no copy is in flight when the CTA ends
            for (uint32_t s = 0; s < kPacked; ++s) landed(full + 8 * s, s < stage ? phase : phase ^ 1u);
        } else if (warp == (uint32_t)kMmaWarp) {
            // ---------------- MMAs ----------------
            uint32_t slot = 0, phase = 0, tile = 0, unitNo = 0;  // tile: key tiles so far (its S buffer, the barriers' parities)
            bool ok = true;
            Walk w = firstWalk;
            const uint32_t idescS = idesc_f16(kTileKeys, false), idescO = idesc_f16(DIM, true);
            auto scores = [&](uint32_t n) {  // S of the n-th tile, from the slot that is next
                if (!wait_warp<false>(barTile + 8 * slot, phase, &abortFlag)) return false;
                tc_fence_after();
                const uint64_t desc = desc_sw128(slots + slot * kSlot, 16);
                const uint32_t d = tmem + kColS + n % kBuffers * kTileKeys;
                if (elect_one()) {
#pragma unroll
                    for (uint32_t k = 0; k < DIM / 16; ++k)
                        mma_a_tmem(d, tmem + kColQ + 8 * k, desc + (k / 4) * (kTileKeys * 128 >> 4) + 2 * (k % 4), idescS, k != 0);
                    commit(barTileFree + 8 * slot);
                    commit(barS + 8 * (n % kBuffers));
                }
                __syncwarp();
                if (++slot == kSlots) slot = 0, phase ^= 1u;
                return true;
            };
            for (bool more = firstMore; more && ok; more = ok && next_segment(w)) {
                ok = wait_warp<false>(barQ, unitNo & 1u, &abortFlag);
                tc_fence_after();
                for (uint32_t i = 0; i < min(kAhead, w.count) && ok; ++i) ok = scores(tile + i);
                for (uint32_t i = 0; i < w.count && ok; ++i, ++tile) {
                    if (!(ok = wait_warp<false>(barTile + 8 * slot, phase, &abortFlag))) break;
                    if (!(ok = wait_warp<false>(barP + 16 * (tile % kBuffers), tile / kBuffers & 1u, &abortFlag))) break;
                    tc_fence_after();
                    const uint64_t desc = desc_sw128(slots + slot * kSlot, kTileKeys * 128);
                    const uint32_t p = tmem + kColS + tile % kBuffers * kTileKeys;
                    if (elect_one()) {
#pragma unroll
                        for (uint32_t k = 0; k < kTileKeys / 32; ++k) mma_a_tmem(tmem + kColO, p + 8 * k, desc + k * (2048 >> 4), idescO, (i | k) != 0);
                    }
                    __syncwarp();
                    if (!(ok = wait_warp<false>(barP + 16 * (tile % kBuffers) + 8, tile / kBuffers & 1u, &abortFlag))) break;
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (uint32_t k = kTileKeys / 32; k < kTileKeys / 16; ++k) mma_a_tmem(tmem + kColO, p + 8 * k, desc + k * (2048 >> 4), idescO, 1u);
                        commit(barTileFree + 8 * slot);
                        commit(barO + 8 * (tile % kBuffers));
                        commit(barInfoFree + 8 * (tile % kInfo));  // weights formed, values expanded: nobody looks at the tile's scales any more
                    }
                    __syncwarp();
                    if (++slot == kSlots) slot = 0, phase ^= 1u;
                    if (i + kAhead < w.count) ok = scores(tile + kAhead);
                }
                ++unitNo;
            }
            // nor any product, when tensor memory goes back
            if (elect_one()) commit(barDone);
            __syncwarp();
            landed(barDone, 0);
        } else if (warp == (uint32_t)kScaleWarp) {
            // ---------------- scales: a lane two neighbouring keys of a tile ----------------
            // What no row sees is nothing; a visible key with a value (or a value of its value) that is no number is NaN, its value
            // nothing; keys whose page is outside the cache are marked.  A group's word for the expansion: f16 scale * 2^(24 - E) | f16 bias * 2^-E, the largest of
            // 16 scale and |bias| of the tile 2^-6 .. 2^-5.
            uint32_t tile = 0;
            bool ok = true;
            Walk w = firstWalk;
            for (bool more = firstMore; more && ok; more = ok && next_segment(w)) {
                // Of values far below (2^-64) the largest of the segment so far, or of zeros, the tile's own power would put M so far above its
                // logits that its weights fell out of 32 bits, and out of the sum.
                int floorV = -100;
                const int pLast = w.q.p0 + (int)w.q.tokens - 1;
                for (uint32_t i = 0; i < w.count; ++i, ++tile) {
                    const uint32_t at = tile % kPacked, info = tile % kInfo;
                    const int j0 = (int)key_at(w.q, w.t0 + i);
                    if (!(ok = wait_warp<true>(barPack + 8 * at, tile / kPacked & 1u, &abortFlag))) break;
                    // keys that some row does not see, or on a page outside the cache
                    const uint32_t gone = holes[at] & ((1u << pieces) - 1u);
                    const bool unseen = gone || j0 + (int)kTileKeys - 1 > w.q.p0 || (a.window && (long long)j0 <= (long long)pLast - a.window && (uint32_t)j0 + kTileKeys > a.sinks);
                    uint32_t v[2][2][NG];  // [keys, values][the lane's key][group]
                    const uint32_t key0 = 2 * lane, from = words + at * words_bytes(DIM) + (((key0 >> args.pieceShift) * 2) << args.pieceShift) * WB + (key0 & (pieceKeys - 1u)) * WB;  // of a piece: keys' words, then values'
                    uint32_t most[2] = {0u, 0u};  // magnitudes of scales and biases
#pragma unroll
                    for (int side = 0; side < 2; ++side)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            lds_words<NG>(from + ((side << args.pieceShift) + h) * WB, v[side][h]);
#pragma unroll
                            for (int G = 0; G < NG; ++G) most[side] = __vmaxu2(most[side], v[side][h][G] & 0x7FFF7FFFu);
                        }
                    auto none = [](uint32_t m) { return max(m & 0xFFFFu, m >> 16) >= 0x7F80u; };
                    uint32_t out[2] = {0u, 0u};  // bit l: key 2 l, key 2 l + 1
                    if (__any_sync(0xFFFFFFFFu, unseen || none(most[0]) || none(most[1]))) {
                        most[0] = most[1] = 0u;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int j = j0 + (int)key0 + h, p = max(j, w.q.p0);  // of the rows that may see it, the one whose window goes back furthest
                            const bool hole = gone >> (key0 >> args.pieceShift) & 1u;
                            const bool seen = p <= pLast && (!a.window || (long long)j > (long long)p - a.window || (uint32_t)j < a.sinks);
                            bool broke = false;
#pragma unroll
                            for (int side = 0; side < 2; ++side)
#pragma unroll
                                for (int G = 0; G < NG; ++G) broke |= is_broken(v[side][h][G]);
                            out[h] = __ballot_sync(0xFFFFFFFFu, seen && hole);
#pragma unroll
                            for (int side = 0; side < 2; ++side)
#pragma unroll
                                for (int G = 0; G < NG; ++G) {
                                    if (!seen || hole || broke) v[side][h][G] = 0u;
                                    most[side] = __vmaxu2(most[side], v[side][h][G] & 0x7FFF7FFFu);
                                }
                            // (the key of either makes its column of S NaN, which only rows that see it take)
                            if (seen && !hole && broke)
#pragma unroll
                                for (int G = 0; G < NG; ++G) v[0][h][G] = 0x7FC07FC0u;
                        }
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(barPackFree + 8 * at);
                    int exponent[2];
#pragma unroll
                    for (int side = 0; side < 2; ++side) {
                        const uint32_t largest = __reduce_max_sync(0xFFFFFFFFu, max(((most[side] & 0xFFFFu) >> 7) + 4u, most[side] >> 23));
                        exponent[side] = min(max((int)largest - 127 + 6, side ? floorV : -100), 120);
                    }
                    floorV = max(floorV, exponent[1] - 64);
                    if (!(ok = wait_warp<true>(barInfoFree + 8 * info, tile / kInfo & 1u ^ 1u, &abortFlag))) break;
#pragma unroll
                    for (int side = 0; side < 2; ++side) {
                        const float toBias = power_of_two(-exponent[side]), toScale = power_of_two(24 - exponent[side]);
#pragma unroll
                        for (int G = 0; G < NG; ++G)
                            sts64(scales + info * words_bytes(DIM) + side * kWordSide + (G * kTileKeys + key0) * 4, pack_f16(low16(v[side][0][G]) * toScale, high16(v[side][0][G]) * toBias),
                                  pack_f16(low16(v[side][1][G]) * toScale, high16(v[side][1][G]) * toBias));
                    }
                    __syncwarp();
                    if (lane == 0) {
                        tileInfo[info] = make_float4(power_of_two(exponent[0]), (float)exponent[1], unseen ? 1.0f : 0.0f, 0.0f);
                        hidden[info][0] = out[0], hidden[info][1] = out[1];
                        mbar_arrive(barInfo + 8 * info);
                    }
                }
            }
        } else if (warp >= (uint32_t)kFirstDequant) {
            // ---------------- expansion: the groups of warps take slots K0, K1, (K2,) V0, K2 (K3), V1, ... in turn ----------------
            const uint32_t dw = warp - kFirstDequant, grp = dw / kGroupWarps, inGroup = dw % kGroupWarps;
            uint32_t item = 0, tile = 0;  // slots filled by all groups; key tiles so far
            bool ok = true;
            auto fill = [&](uint32_t n, uint32_t side) {  // keys or values of the CTA's n-th tile
                const uint32_t slot = item % kSlots, slotPhase = item / kSlots & 1u, pack = n % kPacked + side * kPacked, packPhase = n / kPacked & 1u, info = n % kInfo;
                // The slot before the codes: it is free when the item kSlots before this one has been multiplied, and with it the
                // values that lay in this place of the packed ring before.  Waiting for the codes first, a group that is ahead of the one
                // that expands those (copies land in any order) would take the parity of the round before last for its own.
                // (A lane that gives up goes on with what lies there, so that the warp ends the item as one.)
                bool mine = wait_lane<false>(barInfo + 8 * info, n / kInfo & 1u, &abortFlag);
                mine = mine && wait_lane<false>(barTileFree + 8 * slot, slotPhase ^ 1u, &abortFlag) && wait_lane<false>(barPack + 8 * pack, packPhase, &abortFlag);
#pragma unroll 1
                for (uint32_t e = 0; e < kUnitsEach; ++e) {
                    const uint32_t unit = e * (32 * kGroupWarps) + inGroup * 32 + lane, key = unit % kTileKeys, G = unit / kTileKeys;
                    const uint32_t word = lds32(scales + info * words_bytes(DIM) + side * kWordSide + unit * 4);
                    const uint32_t from = packed + pack * kPack + key * CB;
                    const uint4 v[2] = {lds128(from + ((G * 32) ^ chunk_flip<DIM>(key))), lds128(from + ((G * 32 + 16) ^ chunk_flip<DIM>(key)))};
                    const uint32_t s0 = __byte_perm(word, word, 0x1010), bb = __byte_perm(word, word, 0x3232), s1 = mul_f16x2(s0, 0x2C002C00u);  // 2^-4
                    const uint32_t to = slots + slot * kSlot + G * (kTileKeys * 128) + key * 128;
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h) {
                        // Four runs of eight values; a chunk is their values n and n + 4.  (In this order four lanes hold a row of
                        // 32 values in tensor memory, a run each: queries come, and outputs go, 64 bytes of a row at a time.)
                        const uint32_t c[4] = {v[h].x, v[h].y, v[h].z, v[h].w};
                        const uint32_t upper[4] = {c[0] >> 8, c[1] >> 8, c[2] >> 8, c[3] >> 8};
#pragma unroll
                        for (uint32_t n = 0; n < 4; ++n) {
                            const uint32_t *w4 = n < 2 ? c : upper, mask = n % 2 ? 0x00F000F0u : 0x000F000Fu, scale = n % 2 ? s1 : s0;
                            sts128(to + (((4 * h + n) ^ (key & 7u)) << 4), fma_f16x2(w4[0] & mask, scale, bb), fma_f16x2(w4[1] & mask, scale, bb),
                                   fma_f16x2(w4[2] & mask, scale, bb), fma_f16x2(w4[3] & mask, scale, bb));
                        }
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                ok = __all_sync(0xFFFFFFFFu, mine);
                if (lane == 0 && ok) {
                    mbar_arrive(barPackFree + 8 * pack);
                    mbar_arrive(barTile + 8 * slot);
                }
            };
            Walk w = firstWalk;
            for (bool more = firstMore; more && ok; more = ok && next_segment(w)) {
                // a segment of n tiles is 2 n slots: the keys of the first kAhead, then for every tile i its values and the keys of i + kAhead
                const uint32_t lead = min(kAhead, w.count), paired = lead + 2 * (w.count - lead);
                for (uint32_t k = 0; k < 2 * w.count && ok; ++k, ++item) {
                    if (item % kGroups != grp) continue;
                    const bool isKey = k < lead || (k < paired && ((k - lead) & 1u));
                    fill(tile + (k < lead ? k : k < paired ? (k - lead) / 2 + (isKey ? lead : 0u) : k - w.count), isKey ? 0u : 1u);
                }
                tile += w.count;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsRows));
        if (begin < end) {
            // ---------------- rows ----------------
            const uint32_t wg = (warp - kFirstRowWarp) / 4, quarter = warp & 3u, row = quarter * 32 + lane;
            const uint32_t lanes = (quarter * 32) << 16;
            uint32_t tile = 0, joins = 0;
            bool ok = true;
            [[maybe_unused]] uint4 firstPart = make_uint4(0u, 0u, 0u, 0u);  // prefix: of the run's last unit, where others have the rest
            uint32_t mineRows[4];  // token << 16 | head of the rows lane / 4 + 8 k of the warp's 32
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t r = quarter * 32 + 8 * k + (lane >> 2);
                mineRows[k] = (r / group) << 16 | r % group;
            }
            Walk w = firstWalk;
            for (bool more = firstMore; more && ok; more = ok && next_segment(w)) {
                const uint32_t token = row / group;
                const bool there = token < w.q.tokens;
                const int p = w.q.p0 + (int)token;
                auto meet = [&] {  // of both warpgroups
                    __syncwarp();
                    if (lane == 0) mbar_arrive(barJoin);
                    ok = wait_warp<false>(barJoin, joins++ & 1u, &abortFlag);
                    return ok;
                };
                // queries: f16 at a power of two of the row's largest value; either warpgroup half of a row, all its loads in flight,
                // four lanes a row of 64 bytes
                float toLog2;
                {
                    constexpr int kBlocks = DIM / 64;  // of 32 values in half a row
                    uint4 v[4][kBlocks];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t tok = mineRows[k] >> 16;
                        const uint4 *src = reinterpret_cast<const uint4 *>(a.q + (size_t)(w.q.firstRow + tok) * a.qStride + (w.head * group + (mineRows[k] & 0xFFFFu)) * DIM + wg * (DIM / 2)) + (lane & 3u);
#pragma unroll
                        for (int i = 0; i < kBlocks; ++i) v[k][i] = tok < w.q.tokens ? __ldg(src + 4 * i) : make_uint4(0u, 0u, 0u, 0u);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t largest = 0;
#pragma unroll
                        for (int i = 0; i < kBlocks; ++i)
                            largest = __vmaxu2(largest, __vmaxu2(__vmaxu2(v[k][i].x & 0x7FFF7FFFu, v[k][i].y & 0x7FFF7FFFu), __vmaxu2(v[k][i].z & 0x7FFF7FFFu, v[k][i].w & 0x7FFF7FFFu)));
                        largest = __vmaxu2(largest, __shfl_xor_sync(0xFFFFFFFFu, largest, 1));
                        largest = __vmaxu2(largest, __shfl_xor_sync(0xFFFFFFFFu, largest, 2));
                        if ((lane & 3u) == 0u) largestShared[wg][quarter * 32 + 8 * k + (lane >> 2)] = max(largest & 0xFFFFu, largest >> 16) >> 7;
                    }
                    if (!meet()) break;
                    auto exponent_of = [&](uint32_t r) { return max(max(largestShared[0][r], largestShared[1][r]), 7u); };
                    toLog2 = logit_factor(a.scale, (int)exponent_of(row) - 134);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        float down[2];
#pragma unroll
                        for (int k = 0; k < 2; ++k) down[k] = __uint_as_float((261u - exponent_of(quarter * 32 + 16 * half + 8 * k + (lane >> 2))) << 23);  // the largest is 2^7 .. 2^8
#pragma unroll
                        for (int i = 0; i < kBlocks; ++i) {
                            uint32_t o[8];  // columns 4 j + lane % 4 of rows lane / 4 and lane / 4 + 8
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const uint4 u = v[2 * half + k][i];
                                o[k] = pack_f16(low16(u.x) * down[k], low16(u.z) * down[k]);
                                o[2 + k] = pack_f16(high16(u.x) * down[k], high16(u.z) * down[k]);
                                o[4 + k] = pack_f16(low16(u.y) * down[k], low16(u.w) * down[k]);
                                o[6 + k] = pack_f16(high16(u.y) * down[k], high16(u.w) * down[k]);
                            }
                            tc_store_16x16(tmem + lanes + (half << 20) + kColQ + wg * (DIM / 4) + 16 * i, o);
                        }
                    }
                    tc_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(barQ);
                }
                float ref = kNone, sum = 0.0f;  // the warpgroup's part of the weights' sum, at 2^ref, its largest logit
                uint32_t i = (tile ^ wg) & 1u;  // the segment's first tile of this warpgroup
                for (tile += i; i < w.count; i += 2, tile += 2) {
                    const uint32_t info = tile % kInfo;
                    if (!(ok = wait_warp<false>(barS + 8 * (tile % kBuffers), tile / kBuffers & 1u, &abortFlag))) break;
                    tc_fence_after();
                    const uint32_t s0 = tmem + lanes + kColS + tile % kBuffers * kTileKeys;
                    uint32_t lo[32], hi[32];
                    tc_load_32cols(s0, lo);
                    tc_load_32cols(s0 + 32, hi);
                    const float4 about = tileInfo[info];  // 2^eK, eV, whether some row does not see some key
                    tc_wait_ld();
                    float *s = reinterpret_cast<float *>(lo), *u = reinterpret_cast<float *>(hi);
                    if (about.z != 0.0f) {
                        // the keys that the row sees: up to its own, and above the window's end or below the last sink
                        const uint32_t gone0 = hidden[info][0], gone1 = hidden[info][1];
                        const long long j0 = key_at(w.q, w.t0 + i);
                        unsigned long long sees = first_bits(p - j0 + 1);
                        if (a.window) sees &= ~first_bits(p - j0 - a.window + 1) | first_bits((long long)a.sinks - j0);
                        if (gone0 | gone1) sees &= ~(spread_bits(gone0) | spread_bits(gone1) << 1);
                        const uint32_t sees0 = (uint32_t)sees, sees1 = (uint32_t)(sees >> 32);
#pragma unroll
                        for (int c = 0; c < 32; ++c) {
                            s[c] = sees0 >> c & 1u ? s[c] : -INFINITY;
                            u[c] = sees1 >> c & 1u ? u[c] : -INFINITY;
                        }
                    }
                    float most[4] = {s[0], s[1], u[0], u[1]};
#pragma unroll
                    for (int c = 2; c < 32; c += 4) {
                        most[0] = fmaxf(fmaxf(most[0], s[c]), s[c + 2 < 32 ? c + 2 : c]);
                        most[1] = fmaxf(fmaxf(most[1], s[c + 1]), s[c + 3 < 32 ? c + 3 : c + 1]);
                        most[2] = fmaxf(fmaxf(most[2], u[c]), u[c + 2 < 32 ? c + 2 : c]);
                        most[3] = fmaxf(fmaxf(most[3], u[c + 1]), u[c + 3 < 32 ? c + 3 : c + 1]);
                    }
                    const float f = fmaxf(toLog2 * about.x, 0x1p-126f), product = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
                    const float peak = fmaf(product, f, about.y), level = fmaxf(ref, product * f);
                    // the maximum that the tile before settled on
                    float top = kNone;
                    if (i) {
                        if (!(ok = wait_warp<false>(barTop + 8 * ((wg ^ 1u) * 4 + quarter), (tile - 1) >> 1 & 1u, &abortFlag))) break;
                        top = topShared[row];
                    }
                    if (__any_sync(0xFFFFFFFFu, peak > top + kLazy)) {
                        const float next = fmaxf(top, peak), down = exp2_fast(top - next);
                        top = next;
                        if (i) {  // O so far, once the products in flight are done
                            if (!(ok = wait_warp<false>(barO + 8 * ((tile - 1) % kBuffers), (tile - 1) / kBuffers & 1u, &abortFlag))) break;
                            tc_fence_after();
#pragma unroll 1
                            for (uint32_t c = 0; c < DIM; c += 16) {
                                uint32_t v[16];
                                tc_load_16cols(tmem + lanes + kColO + c, v);
                                tc_wait_ld();
#pragma unroll
                                for (int k = 0; k < 16; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * down);
                                tc_store_16cols(tmem + lanes + kColO + c, v);
                            }
                            tc_wait_st();
                        }
                    }
                    topShared[row] = top;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(barTop + 8 * (wg * 4 + quarter));
                    sum *= exp2_fast(ref - level);
                    ref = level;
                    const float shift = about.y - top + kWeightScale;
                    const unsigned long long f2 = pair_f32(f, f), shift2 = pair_f32(shift, shift);
                    unsigned long long part = pair_f32(0.0f, 0.0f), part2 = part;
                    auto weigh = [&](const float *v, uint32_t to) {  // 32 logits: weights to 16 columns
                        uint32_t o[16];
#pragma unroll
                        for (int c = 0; c < 32; c += 4) {
                            const unsigned long long x = fma_f32x2(pair_f32(v[c], v[c + 1]), f2, shift2), y = fma_f32x2(pair_f32(v[c + 2], v[c + 3]), f2, shift2);
                            const float x0 = exp2_fast(first_f32(x)), x1 = exp2_fast(second_f32(x)), y0 = exp2_fast(first_f32(y)), y1 = exp2_fast(second_f32(y));
                            part = add_f32x2(part, pair_f32(x0, x1));
                            part2 = add_f32x2(part2, pair_f32(y0, y1));
                            o[c / 2] = pack_f16(x0, x1);
                            o[c / 2 + 1] = pack_f16(y0, y1);
                        }
                        tc_store_16cols(to, o);
                    };
                    weigh(s, s0);
                    tc_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(barP + 16 * (tile % kBuffers));  // (the products of the first 32 keys may begin)
                    weigh(u, s0 + 16);
                    part = add_f32x2(part, part2);
                    // (A weight is 2^(S f + eV - M) here.  M is at most 72 above the largest logit plus eV; where it is further above this warpgroup's,
                    // the other has far larger ones.  M and the logit first: their difference is exact, as P's rounding of M takes it.)
                    sum = fmaf(first_f32(part) + second_f32(part), exp2_fast(fminf((top - level) - about.y, 120.0f)), sum);
                    tc_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(barP + 16 * (tile % kBuffers) + 8);
                }
                if (!ok) break;
                tile = tile - i + w.count;

                // ---- the unit's rows, or this CTA's part of them: either warpgroup every second 32 values ----
                sumShared[wg][row] = sum;
                refShared[wg][row] = ref;
                if (!meet() || !(ok = wait_warp<false>(barO + 8 * ((tile - 1) % kBuffers), (tile - 1) / kBuffers & 1u, &abortFlag))) break;
                tc_fence_after();
                if constexpr (kSuffix) pdl_wait();  // (for what the prefixes gave, and the parts' memory)
                const float top = topShared[row];
                const float largest = fmaxf(refShared[0][row], refShared[1][row]);
                sum = sumShared[0][row] * exp2_fast(refShared[0][row] - largest) + sumShared[1][row] * exp2_fast(refShared[1][row] - largest);
                const bool whole = w.count == w.q.tiles;
                const uint32_t part = 2 * cta + (w.t0 == 0 ? 1u : 0u);
                float factor = sum == 0.0f ? 0.0f : exp2_fast(top - largest) / sum;  // (-108 .. 120, of the values' powers)
                // a row's place among those of the prefix, and the first of its values there
                auto shared_place = [&](uint32_t token, uint32_t h) { return (size_t)(w.q.firstRow + token) * a.heads + w.head * group + h; };
                // what the prefix gives the row's result, and what the row's own part keeps; the sums there are of the weights themselves
                constexpr float kUnweight = 1.0f / (1u << (int)kWeightScale);
                auto join_prefix = [&](size_t place, float level, float weights, float &keep) {
                    weights *= kUnweight;
                    const float2 st = __ldcg(a.shared.stats + place);
                    const float most = fmaxf(level, st.x), mine = exp2_fast(level - most), other = st.y * exp2_fast(st.x - most), all = fmaf(weights, mine, other);
                    keep = weights == 0.0f || all == 0.0f ? 0.0f : weights * mine / all;
                    return all == 0.0f ? 0.0f : other / all;
                };
                float given = 0.0f;
                if constexpr (kPrefix) {
                    if (whole && there && wg == 0) a.shared.stats[shared_place(token, row % group)] = make_float2(largest, sum * kUnweight);
                }
                if constexpr (kSuffix) {
                    if (whole && there && w.q.joins) {
                        float keep;
                        given = join_prefix(shared_place(token, row % group), largest, sum, keep);
                        factor *= keep;
                    }
                }
                if (whole) {
                    // four lanes 64 bytes of a row
                    float factors[4];
                    uint16_t *to[4];
                    [[maybe_unused]] float gives[4];
                    [[maybe_unused]] float *shared[4];
                    if constexpr (kPrefix || kSuffix) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            gives[k] = __shfl_sync(0xFFFFFFFFu, given, 8 * k + (lane >> 2));
                            shared[k] = a.shared.values + shared_place(mineRows[k] >> 16, mineRows[k] & 0xFFFFu) * DIM + 8 * (lane & 3u);
                        }
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        factors[k] = __shfl_sync(0xFFFFFFFFu, factor, 8 * k + (lane >> 2));
                        to[k] = a.out + (size_t)(w.q.firstRow + (mineRows[k] >> 16)) * a.outStride + (w.head * group + (mineRows[k] & 0xFFFFu)) * DIM + 8 * (lane & 3u);
                    }
#pragma unroll 1
                    for (uint32_t c = 32 * wg; c < DIM; c += 32 * kRowGroups) {
                        uint32_t o[2][16];
                        tc_load_16x32(tmem + lanes + kColO + c, o[0]);
                        tc_load_16x32(tmem + lanes + (1u << 20) + kColO + c, o[1]);
                        tc_wait_ld();
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t *u = o[k >> 1] + 2 * (k & 1);  // u[4 j], u[4 j + 1]: values j and j + 4 of the lane's run
                            auto at = [&](int n) { return __uint_as_float(u[4 * (n & 3) + (n >> 2)]) * factors[k]; };
                            if ((mineRows[k] >> 16) < w.q.tokens) {
                                if constexpr (kPrefix) {
                                    *reinterpret_cast<float4 *>(shared[k] + c) = make_float4(at(0), at(1), at(2), at(3));
                                    *reinterpret_cast<float4 *>(shared[k] + c + 4) = make_float4(at(4), at(5), at(6), at(7));
                                    continue;
                                } else if constexpr (kSuffix) {
                                    if (w.q.joins) {
                                        const float4 x = __ldcg(reinterpret_cast<const float4 *>(shared[k] + c)), y = __ldcg(reinterpret_cast<const float4 *>(shared[k] + c + 4));
                                        const float g = gives[k];
                                        *reinterpret_cast<uint4 *>(to[k] + c) = make_uint4(pack_bf16x2(fmaf(x.x, g, at(0)), fmaf(x.y, g, at(1))), pack_bf16x2(fmaf(x.z, g, at(2)), fmaf(x.w, g, at(3))),
                                                                                           pack_bf16x2(fmaf(y.x, g, at(4)), fmaf(y.y, g, at(5))), pack_bf16x2(fmaf(y.z, g, at(6)), fmaf(y.w, g, at(7))));
                                        continue;
                                    }
                                }
                                *reinterpret_cast<uint4 *>(to[k] + c) = make_uint4(pack_bf16x2(at(0), at(1)), pack_bf16x2(at(2), at(3)), pack_bf16x2(at(4), at(5)), pack_bf16x2(at(6), at(7)));
                            }
                        }
                    }
                } else {
                    // (a part's values, four of a row behind four of the next, in the order of O's columns)
#pragma unroll 1
                    for (uint32_t c = 32 * wg; c < DIM; c += 32 * kRowGroups) {
                        uint32_t o[32];
                        tc_load_32cols(tmem + lanes + kColO + c, o);
                        tc_wait_ld();
                        float4 *at = reinterpret_cast<float4 *>(args.partials) + ((size_t)part * (DIM / 4) + c / 4) * kRows + row;
                        if (there)
#pragma unroll
                            for (int k = 0; k < 8; ++k) at[k * kRows] = make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]), __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3]));
                    }
                }
                tc_fence_before();  // (the next unit's products overwrite O once both warpgroups have brought their queries)
                if (!whole) {
                    if (there && wg == 0) args.stats[part * kRows + row] = make_float4(top, largest, sum, 0.0f);
                    const uint32_t c0 = cta_of(w.first + kUnitCost), c1 = cta_of(w.first + kUnitCost + w.q.tiles - 1), parts = c1 - c0 + 1;
                    if constexpr (kPrefix) {  // (joined by a launch of their own: the last to arrive would take 13 us for ten)
                        if (w.t0 == 0) firstPart = make_uint4(w.q.firstRow, w.q.tokens, w.head, parts);
                        if (!meet()) break;
                        continue;
                    }
                    // whether this is the last of `expected` CTAs; then what they wrote is there
                    auto arrive = [&](uint32_t *counter, uint32_t expected) {
                        if (!meet()) return false;
                        if (wg == 0 && row == 0) {
                            __threadfence();  // (cumulative: for the parts that the barrier made this thread see)
                            const uint32_t n = atomicAdd(counter, 1u);
                            __threadfence();
                            lastPart = n == expected - 1;
                            if (n == expected - 1) *counter = 0u;
                        }
                        return meet() && lastPart != 0u;
                    };
                    // parts of CTAs from, from + step, ... joined, into the unit's rows or the first one's place: a warp 32 rows and
                    // 32 of their values at a time, two parts' loads in flight
                    auto join = [&](uint32_t from, uint32_t count, uint32_t step, bool last) {
                        auto part_of = [&](uint32_t c) { return 2 * c + (c == c0 ? 1u : 0u); };
                        constexpr uint32_t kAtOnce = 2, kValues = 4;
                        const uint32_t used = w.q.tokens * group, blocks = (used + 31) / 32;
#pragma unroll 1
                        for (uint32_t item = warp - kFirstRowWarp; item < blocks * (DIM / 8 / kValues); item += kRowWarps) {
                            const uint32_t mine = item % blocks * 32 + lane, d = item / blocks * (8 * kValues);
                            if (mine >= used) continue;
                            float all = kNone, level = kNone, weights = 0.0f, v[8 * kValues];
#pragma unroll
                            for (uint32_t k = 0; k < 8 * kValues; ++k) v[k] = 0.0f;
                            auto place = [&](uint32_t n) { return reinterpret_cast<float4 *>(args.partials) + ((size_t)n * (DIM / 4) + d / 4) * kRows + mine; };
#pragma unroll 1
                            for (uint32_t k0 = 0; k0 < count; k0 += kAtOnce) {
                                float4 st[kAtOnce], t[kAtOnce][2 * kValues];
#pragma unroll
                                for (uint32_t k = 0; k < kAtOnce; ++k) {
                                    const uint32_t n = part_of(from + min(k0 + k, count - 1) * step);
                                    st[k] = __ldcg(args.stats + n * kRows + mine);
#pragma unroll
                                    for (uint32_t h = 0; h < 2 * kValues; ++h) t[k][h] = __ldcg(place(n) + h * kRows);
                                }
                                float next = all, nextLevel = level;
#pragma unroll
                                for (uint32_t k = 0; k < kAtOnce; ++k) next = fmaxf(next, st[k].x), nextLevel = fmaxf(nextLevel, st[k].y);
                                const float keep = exp2_fast(all - next);
                                weights *= exp2_fast(level - nextLevel);
                                all = next, level = nextLevel;
#pragma unroll
                                for (uint32_t k = 0; k < 8 * kValues; ++k) v[k] *= keep;
#pragma unroll
                                for (uint32_t k = 0; k < kAtOnce; ++k) {
                                    if (k0 + k >= count) break;
                                    const float g = exp2_fast(st[k].x - all);
                                    weights = fmaf(st[k].z, exp2_fast(st[k].y - level), weights);
#pragma unroll
                                    for (uint32_t h = 0; h < 2 * kValues; ++h) {
                                        v[4 * h] = fmaf(t[k][h].x, g, v[4 * h]), v[4 * h + 1] = fmaf(t[k][h].y, g, v[4 * h + 1]);
                                        v[4 * h + 2] = fmaf(t[k][h].z, g, v[4 * h + 2]), v[4 * h + 3] = fmaf(t[k][h].w, g, v[4 * h + 3]);
                                    }
                                }
                            }
                            if (last) {
                                float f = weights == 0.0f ? 0.0f : exp2_fast(all - level) / weights;
                                if constexpr (kSuffix) {
                                    const size_t place = shared_place(mine / group, mine % group);
                                    const float *values = a.shared.values + place * DIM + d;
                                    if (w.q.joins) {
                                        float keep;
                                        const float g = join_prefix(place, level, weights, keep);
                                        f *= keep;
#pragma unroll
                                        for (uint32_t k = 0; k < 4; ++k) {
                                            const float4 x = __ldcg(reinterpret_cast<const float4 *>(values + 8 * k)), y = __ldcg(reinterpret_cast<const float4 *>(values + 8 * k + 4));
                                            v[2 * k] = fmaf(v[2 * k], f, x.x * g), v[8 + 2 * k] = fmaf(v[8 + 2 * k], f, x.y * g);
                                            v[16 + 2 * k] = fmaf(v[16 + 2 * k], f, x.z * g), v[24 + 2 * k] = fmaf(v[24 + 2 * k], f, x.w * g);
                                            v[2 * k + 1] = fmaf(v[2 * k + 1], f, y.x * g), v[9 + 2 * k] = fmaf(v[9 + 2 * k], f, y.y * g);
                                            v[17 + 2 * k] = fmaf(v[17 + 2 * k], f, y.z * g), v[25 + 2 * k] = fmaf(v[25 + 2 * k], f, y.w * g);
                                        }
                                        f = 1.0f;
                                    }
                                }
                                uint16_t *to = a.out + (size_t)(w.q.firstRow + mine / group) * a.outStride + (w.head * group + mine % group) * DIM + d;
#pragma unroll
                                for (uint32_t k = 0; k < 4; ++k)  // value n of run k: column 8 (n % 4) + 2 k + n / 4
                                    *reinterpret_cast<uint4 *>(to + 8 * k) = make_uint4(pack_bf16x2(v[2 * k] * f, v[8 + 2 * k] * f), pack_bf16x2(v[16 + 2 * k] * f, v[24 + 2 * k] * f),
                                                                                        pack_bf16x2(v[2 * k + 1] * f, v[9 + 2 * k] * f), pack_bf16x2(v[17 + 2 * k] * f, v[25 + 2 * k] * f));
                            } else {
#pragma unroll
                                for (uint32_t h = 0; h < 2 * kValues; ++h) place(part_of(from))[h * kRows] = make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
                                if (d == 0) topShared[mine] = all, refShared[0][mine] = level, sumShared[0][mine] = weights;
                            }
                        }
                        if (last || !meet()) return;  // (the first one's maxima have been read)
                        if (wg == 0 && row < used) args.stats[part_of(from) * kRows + row] = make_float4(topShared[row], refShared[0][row], sumShared[0][row], 0.0f);
                    };
                    // by groups of 16 first where there are more (a CTA is the first of one unit and inside another at most: a
                    // group's counter goes by which)
                    constexpr uint32_t kGroupParts = 16;
                    const uint32_t groups = (parts + kGroupParts - 1) / kGroupParts, group0 = c0 + (cta - c0) / kGroupParts * kGroupParts;
                    bool last = groups == 1;
                    uint32_t *counter = args.arrived + (last ? 0 : group0 == c0 ? 1 : 2) * gridDim.x + group0;
                    uint32_t from = group0, count = min(kGroupParts, c1 - group0 + 1), step = 1;
#pragma unroll 1
                    while (arrive(counter, count)) {
                        join(from, count, step, last);
                        if (last || !ok) break;
                        last = true;
                        counter = args.arrived + c0;
                        from = c0, count = groups, step = kGroupParts;
                    }
                    if (!ok) break;
                }
                if (!meet()) break;  // (before the next unit's words in shared memory)
            }
            if constexpr (kPrefix) {
                if (warp == (uint32_t)kFirstRowWarp && lane == 0) a.shared.parts[cta] = firstPart;
            }
        } else if constexpr (kPrefix) {
            if (warp == (uint32_t)kFirstRowWarp && lane == 0) a.shared.parts[cta] = make_uint4(0u, 0u, 0u, 0u);
        }
    }
    if constexpr (kSuffix) pdl_wait();  // (this launch is not over before the one in front)
    // every role is done, or gave up after a bounded wait; copies and products have landed
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && abortFlag) *a.errorFlag = kFlagWait;
    tc_fence_after();
    if (warp == (uint32_t)kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// The parts of a prefix's units joined, in the CTAs' order: a CTA takes sixteen values of one unit's rows, a thread a row.  Bound by latency:
// four parts' loads in flight (16 units of ten parts 9.5 us by itself; the last CTA to arrive took 13 for its unit, behind all others).
template <int DIM>
__global__ void __launch_bounds__(kTileRows) k_join_prefix(const __grid_constant__ TilesArgs args) {
    constexpr float kUnweight = 1.0f / (1u << (int)kWeightScale);
    constexpr uint32_t kAtOnce = 4;
    const AttendArgs &a = args.a;
    const uint32_t row = threadIdx.x, c0 = blockIdx.x, block = blockIdx.y / 2, half = blockIdx.y % 2, group = a.heads / a.kvHeads;
    pdl_trigger();  // (the successor reads what is older than the launch in front before it waits, and that was complete when this one began)
    pdl_wait();
    const uint4 unit = a.shared.parts[c0];  // first row, rows, head, parts
    if (row >= unit.y * group || unit.w == 0u) return;
    auto slot_of = [&](uint32_t k) { return 2 * (c0 + k) + (k == 0 ? 1u : 0u); };
    float all = kNone, level = kNone, weights = 0.0f, v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = 0.0f;
    for (uint32_t k0 = 0; k0 < unit.w; k0 += kAtOnce) {
        float4 st[kAtOnce], t[kAtOnce][4];
#pragma unroll
        for (uint32_t k = 0; k < kAtOnce; ++k) {
            const uint32_t slot = slot_of(min(k0 + k, unit.w - 1u));
            st[k] = __ldcg(args.stats + slot * kRows + row);
            // columns of the block of 32: four at 4 half + 8 i, values i and i + 4 of runs 2 half and 2 half + 1 of eight
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) t[k][i] = __ldcg(reinterpret_cast<const float4 *>(args.partials) + ((size_t)slot * (DIM / 4) + block * 8 + half + 2 * i) * kRows + row);
        }
        float next = all, nextLevel = level;
#pragma unroll
        for (uint32_t k = 0; k < kAtOnce; ++k) next = fmaxf(next, st[k].x), nextLevel = fmaxf(nextLevel, st[k].y);
        const float keep = exp2_fast(all - next);
        weights *= exp2_fast(level - nextLevel);
        all = next, level = nextLevel;
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] *= keep;
#pragma unroll
        for (uint32_t k = 0; k < kAtOnce; ++k) {
            if (k0 + k >= unit.w) break;
            const float g = exp2_fast(st[k].x - all);
            weights = fmaf(st[k].z, exp2_fast(st[k].y - level), weights);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = fmaf(t[k][i].x, g, v[i]), v[i + 4] = fmaf(t[k][i].y, g, v[i + 4]);
                v[8 + i] = fmaf(t[k][i].z, g, v[8 + i]), v[12 + i] = fmaf(t[k][i].w, g, v[12 + i]);
            }
        }
    }
    const float f = weights == 0.0f ? 0.0f : exp2_fast(all - level) / weights;
    const size_t place = (size_t)(unit.x + row / group) * a.heads + unit.z * group + row % group;
    if (blockIdx.y == 0) a.shared.stats[place] = make_float2(level, weights * kUnweight);
    float4 *to = reinterpret_cast<float4 *>(a.shared.values + place * DIM + block * 32 + half * 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = make_float4(v[4 * i] * f, v[4 * i + 1] * f, v[4 * i + 2] * f, v[4 * i + 3] * f);
}

KernelSmemMemo tilesMemo[3][3];

template <TilesOf OF, int DIM>
bool launch_tiles(FFAttention *att, KernelSmemMemo &memo, const CUtensorMap &codes, const CUtensorMap &words, const TilesArgs &args, cudaStream_t stream, const char **error) {
    if (!memo.prepare(k_attend_tiles<DIM, OF>, att->device, tiles_smem(DIM), kTilesThreads, nullptr, error)) return false;
    return launched(att, launch_pdl(k_attend_tiles<DIM, OF>, dim3(att->smCount), dim3(kTilesThreads), tiles_smem(DIM), stream, codes, words, args), "k_attend_tiles", error) &&
           (OF != TilesOf::kPrefix || launched(att, launch_pdl(k_join_prefix<DIM>, dim3(att->smCount, DIM / 16), dim3(kTileRows), 0, stream, args), "k_join_prefix", error));
}

}  // namespace

template <TilesOf OF>
static bool launch_tiles_of(FFAttention *att, const AttendArgs &a, cudaStream_t stream, const char **error) {
    const uint32_t dim = att->cfg.headDim;
    TilesArgs args{a, att->partials, att->stats, att->arrived, (uint32_t)__builtin_ctz(att->cfg.pageTokens), (uint32_t)__builtin_ctz(std::min(kTileKeys, a.page.pageTokens)), kRows / (a.heads / a.kvHeads)};
    CUtensorMap codes, words;
    if (!make_pages_maps(&codes, &words, a, dim, 1, error)) return false;
    auto &memo = tilesMemo[(int)OF];
    if (dim == 256) return launch_tiles<OF, 256>(att, memo[2], codes, words, args, stream, error);
    if (dim == 128) return launch_tiles<OF, 128>(att, memo[1], codes, words, args, stream, error);
    return launch_tiles<OF, 64>(att, memo[0], codes, words, args, stream, error);
}

bool launch_attend_tiles(FFAttention *att, const AttendArgs &a, cudaStream_t stream, const char **error) { return launch_tiles_of<TilesOf::kRequest>(att, a, stream, error); }
bool launch_attend_prefix_tiles(FFAttention *att, const AttendArgs &a, cudaStream_t stream, const char **error) { return launch_tiles_of<TilesOf::kPrefix>(att, a, stream, error); }
bool launch_attend_suffix_tiles(FFAttention *att, const AttendArgs &a, cudaStream_t stream, const char **error) { return launch_tiles_of<TilesOf::kSuffix>(att, a, stream, error); }

}  // namespace ff

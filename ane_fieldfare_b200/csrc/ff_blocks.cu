// Choosing blocks of 64 keys of the paged INT4 cache: their mean keys, and for every row the blocks whose mean keys its
// queries score highest.
#include <algorithm>

#include "ff_attention_device.cuh"

namespace ff {

namespace {

constexpr uint32_t kBlockShift = 6;
static_assert(kTileKeys == 1u << kBlockShift, "a block is a tile of the attention kernels");
constexpr int kLeastExponent = -60, kMostExponent = 60;  // of a mean's largest value, as far as it is followed

// ---- mean keys -----------------------------------------------------------------------------------

// A warp takes a block of a key/value head, 64 keys of code * scale + bias, 32 codes a lane and load.  Where the scales are no more than 2^6
// and the biases no more than 2^9 apart their sums are exact in 32 bits (a code times a scale has 12 bits, 64 of them 18), and below 2^128 where no
// exponent is above kMostSummed (64 * 15 * 2^118); other blocks are summed in 64 bits, exact unless the scales are 2^35 apart.  Then whole numbers of 2^(e - 6), e the exponent of the largest value: 7 bits and a sign,
// which bf16 holds.  So nothing about a mean depends on the order of sums.
// Bound by issue slots (56 % of them while active) and by the block's own copies: a code takes a logical operation to mask it, half a product and
// half a sum, and a warp waits for its one block in flight.  576 blocks of 8 heads of 256 (45 MB) take 21.5 us from memory, 2.1 TB/s or 32 % of a copy's
// rate, and 17.9 from L2, as right behind a step's appends.  Steps towards it, from L2: 64-bit sums throughout and loads of 8 bytes 29, 32-bit sums
// 23.4, the block by bulk copies into shared memory 20.6, the next one looked up meanwhile 19.4.  A decode step of 64 requests, one of which completes
// a block, 4.8 us: launch and look-up.
constexpr int kMeansThreads = 512;
constexpr uint32_t kMeansWaitLimit = 1u << 20;
constexpr uint32_t kMostSummed = 127 + 117;  // exponent field of the scales and biases that are summed in 32 bits

struct MeansArgs {
    const uint8_t *pages;
    uint32_t pageCount;
    const uint32_t *blockTable;
    uint32_t tableStride, tableKeys;
    const uint32_t *oldLengths, *newLengths;
    uint32_t requests, kvHeads, pageShift;
    PageLayout page;
    uint16_t *means;
    uint32_t *errorFlag;
};

__device__ __forceinline__ unsigned long long pair_f32(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ unsigned long long pair_u32(uint32_t a, uint32_t b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b));
    return r;
}
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
// 32 values a lane, of lanes `lanes` apart up to 32, added up: each round a lane gives half of what it has and takes the other half of its
// partner's; the first values are then the lane's, `at` of those 32 where they begin.
template <int LANES, typename T>
__device__ __forceinline__ uint32_t join_lanes(T (&value)[32]) {
    uint32_t at = 0;
    int half = 16;
#pragma unroll
    for (uint32_t mask = LANES; mask < 32; mask *= 2, half /= 2) {
        const bool upper = threadIdx.x & mask;
        if (upper) at += half;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (i >= half) break;
            const T give = upper ? value[i] : value[i + half], keep = upper ? value[i + half] : value[i];
            value[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, mask);
        }
    }
    return at;
}
__host__ __device__ constexpr uint32_t means_bytes(uint32_t dim) { return kTileKeys * (dim / 2 + dim / 16); }  // of a block's keys

template <int DIM>
__global__ void __launch_bounds__(kMeansThreads) k_block_means(const __grid_constant__ MeansArgs a) {
    constexpr uint32_t CB = DIM / 2, NG = DIM / 64, kLanes = CB / 16, kKeys = 32 / kLanes;  // lanes a key, keys at once
    constexpr int kSteps = kTileKeys / kKeys, kMine = 32 / kKeys;  // turns of a block; values of a mean that are a lane's
    extern __shared__ __align__(16) uint8_t meansSmem[];
    __shared__ __align__(8) uint64_t barriers[kMeansThreads / 32];
    __shared__ uint32_t first[kMeansThreads + 1], warpSums[kMeansThreads / 32];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = (uint32_t)warp_index();
    const uint32_t bar = sm_addr(barriers) + 8 * warp, held = sm_addr(meansSmem) + warp * means_bytes(DIM), heldWords = held + kTileKeys * CB;  // the warp's block
    uint32_t parity = 0;
    if (lane == 0) {
        bar_init(bar, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_enter();

    // blocks that the requests complete, and where each thread's run of requests begins among them
    const uint32_t run = (a.requests + kMeansThreads - 1) / kMeansThreads;
    struct Span {
        uint32_t begin, count;
    };
    auto span_of = [&](uint32_t r) {
        const uint32_t before = __ldg(a.oldLengths + r), after = __ldg(a.newLengths + r);
        Span s{before >> kBlockShift, 0u};
        if (after > before && after > a.tableKeys && blockIdx.x == 0) *a.errorFlag = kFlagTableRow;
        const uint32_t end = min(after, a.tableKeys) >> kBlockShift;
        if (after > before && end > s.begin) s.count = end - s.begin;
        return s;
    };
    const uint32_t r0 = min(tid * run, a.requests), r1 = min(r0 + run, a.requests);
    uint32_t sum = 0;
    for (uint32_t r = r0; r < r1; ++r) sum = add_work(sum, span_of(r).count);
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
    for (uint32_t w = 0; w < kMeansThreads / 32; ++w) {
        if (w < warp) before += warpSums[w];
        total = add_work(total, warpSums[w]);
    }
    if (total == kTooMuch) {  // (the places are nothing then)
        if (blockIdx.x == 0 && tid == 0) *a.errorFlag = kFlagWork;
        return;
    }
    first[tid] = before + scan - sum;
    if (tid == 0) first[kMeansThreads] = total;
    __syncthreads();

    const uint32_t inKey = lane % kLanes, keyLane = lane / kLanes, pieceShift = min(a.pageShift, kBlockShift), pageTokens = 1u << a.pageShift;
    const unsigned long long items = (unsigned long long)total * a.kvHeads, step = (unsigned long long)gridDim.x * (kMeansThreads / 32);
    const uint32_t pieces = kTileKeys >> pieceShift;
    struct Block {
        uint32_t head, key0, page;  // a lane holds the page of one piece
    };
    auto locate = [&](unsigned long long item) {
        Block b{0u, 0u, 0u};
        if (item >= items) return b;
        uint32_t n = divided(item, a.kvHeads), low = 0, high = kMeansThreads;
        b.head = (uint32_t)item - n * a.kvHeads;
        while (high - low > 1) {
            const uint32_t mid = (low + high) >> 1;
            if (first[mid] <= n) low = mid;
            else high = mid;
        }
        n -= first[low];
        uint32_t r = low * run;
        Span s = span_of(r);
        while (n >= s.count) {
            n -= s.count;
            s = span_of(++r);
        }
        b.key0 = (s.begin + n) << kBlockShift;
        if (lane < pieces) b.page = __ldg(a.blockTable + (size_t)r * a.tableStride + ((b.key0 + (lane << pieceShift)) >> a.pageShift));
        return b;
    };
    Block next = locate((unsigned long long)blockIdx.x * (kMeansThreads / 32) + warp);
    for (unsigned long long item = (unsigned long long)blockIdx.x * (kMeansThreads / 32) + warp; item < items; item += step) {
        const uint32_t head = next.head, key0 = next.key0, page = next.page;
        const bool hole = __any_sync(0xFFFFFFFFu, page >= a.pageCount);
        const uint32_t lastPage = __shfl_sync(0xFFFFFFFFu, page, pieces - 1u);
        if (hole && lane == 0) *a.errorFlag = kFlagPage;
        // the block as it lies, piece by piece, into the warp's shared memory
        __syncwarp();  // (the one before has been read)
        const uint32_t at0 = key0 & (pageTokens - 1u);
        if (lane == 0 && !hole) bar_expect(bar, means_bytes(DIM));
        __syncwarp();
        if (lane < pieces && !hole) {
            const uint8_t *block = a.pages + ((size_t)page * a.kvHeads + head) * a.page.blockBytes;
            bulk_copy(held + lane * (CB << pieceShift), block + (size_t)at0 * CB, CB << pieceShift, bar);
            bulk_copy(heldWords + lane * ((NG * 4) << pieceShift), block + a.page.keyWords + (size_t)at0 * (NG * 4), (NG * 4) << pieceShift, bar);
        }
        __syncwarp();
        next = locate(item + step);  // (while the block comes)
        if (!hole) {
            bool there = mbar_try_wait(bar, parity);
#pragma unroll 1
            for (uint32_t i = 0; i < kMeansWaitLimit && !there; ++i) there = mbar_try_wait(bar, parity);
            if (!__all_sync(0xFFFFFFFFu, there)) {
                if (lane == 0) *a.errorFlag = kFlagWait;
                // given up: no copy is in flight when the CTA ends, and no later one takes this one's bytes for its own
#pragma unroll 1
                for (uint32_t i = 0; i < kMeansWaitLimit && !there; ++i) {
                    __nanosleep(40);
                    there = mbar_try_wait(bar, parity);
                }
                break;
            }
            parity ^= 1u;
        }
        // key k * kKeys + keyLane of the block: its word, its codes
        const uint32_t myCodes = held + keyLane * CB + inKey * 16, myWords = heldWords + (keyLane * NG + inKey / (kLanes / NG)) * 4;
        auto word_of = [&](int k) { return hole ? 0u : lds32(myWords + k * (kKeys * NG * 4)); };
        auto codes_of = [&](int k) { return hole ? make_uint4(0u, 0u, 0u, 0u) : lds128(myCodes + k * (kKeys * CB)); };
        // exponents of the scales, of the biases; exact down to numbers that are zero or below the normal ones, which are looked at one by one
        uint32_t most = 0, least = 0xFFu, biasMost = 0, biasLeast = 0xFFu, at;
        {
            uint32_t greatest = 0u, smallest = 0xFFFFFFFFu;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                const uint32_t e = word_of(k) & 0x7F807F80u;
                greatest = __vmaxu2(greatest, e), smallest = __vminu2(smallest, e);
            }
            most = (greatest & 0xFFFFu) >> 7, biasMost = greatest >> 23, least = (smallest & 0xFFFFu) >> 7, biasLeast = smallest >> 23;
            if (__any_sync(0xFFFFFFFFu, least == 0u || biasLeast == 0u)) {
                least = biasLeast = 0xFFu;
#pragma unroll 1
                for (int k = 0; k < kSteps; ++k) {
                    const uint32_t w = word_of(k);
                    if (w & 0x7FFFu) least = min(least, max(w >> 7 & 0xFFu, 1u));
                    if (w & 0x7FFF0000u) biasLeast = min(biasLeast, max(w >> 23 & 0xFFu, 1u));
                }
            }
        }
        most = __reduce_max_sync(0xFFFFFFFFu, most), least = __reduce_min_sync(0xFFFFFFFFu, least);
        biasMost = __reduce_max_sync(0xFFFFFFFFu, biasMost), biasLeast = __reduce_min_sync(0xFFFFFFFFu, biasLeast);
        double mean[kMine], bias = 0.0;
        if (max(most, biasMost) <= kMostSummed && most <= least + 6u && biasMost <= biasLeast + 9u) {
            // Nibbles i and i + 4 of a word, masked in place: 2^23 + 16^i code, less 2^23, times the scale / 16^i; two codes an instruction.
            unsigned long long sums[16];
            float biases = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) sums[i] = pair_f32(0.0f, 0.0f);
            const unsigned long long less = pair_f32(-8388608.0f, -8388608.0f);
#pragma unroll 4
            for (int k = 0; k < kSteps; ++k) {
                const uint32_t w = word_of(k);
                const uint4 four = codes_of(k);
                const uint32_t word[4] = {four.x, four.y, four.z, four.w};
                biases += high16(w);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float down = low16(w) * (i == 0 ? 1.0f : i == 1 ? 0x1p-4f : i == 2 ? 0x1p-8f : 0x1p-12f);
                    const unsigned long long factor = pair_f32(down, down);
                    const uint32_t mask = 15u << (4 * i);
#pragma unroll
                    for (int n = 0; n < 4; ++n)
                        sums[4 * n + i] = fma_f32x2(add_f32x2(pair_u32((word[n] & mask) | 0x4B000000u, (word[n] >> 16 & mask) | 0x4B000000u), less), factor, sums[4 * n + i]);
                }
            }
            float value[32];
#pragma unroll
            for (int i = 0; i < 16; ++i) value[8 * (i / 4) + i % 4] = __uint_as_float((uint32_t)sums[i]), value[8 * (i / 4) + i % 4 + 4] = __uint_as_float((uint32_t)(sums[i] >> 32));
            at = join_lanes<kLanes>(value);
#pragma unroll
            for (uint32_t mask = kLanes; mask < 32; mask *= 2) biases += __shfl_xor_sync(0xFFFFFFFFu, biases, mask);
            bias = biases;
#pragma unroll
            for (int i = 0; i < kMine; ++i) mean[i] = value[i];
        } else {
            double value[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) value[i] = 0.0;
#pragma unroll 1
            for (int k = 0; k < kSteps; ++k) {
                const uint32_t w = word_of(k);
                const uint4 four = codes_of(k);
                const uint32_t word[4] = {four.x, four.y, four.z, four.w};
                const double scale = (double)low16(w);
                bias += (double)high16(w);
#pragma unroll
                for (int i = 0; i < 32; ++i)  // (2^52 + code less 2^52: a conversion takes longer)
                    value[i] = fma(scale, __hiloint2double(0x43300000, (int)(word[i / 8] >> (4 * (i & 7)) & 15u)) - 0x1p52, value[i]);
            }
            at = join_lanes<kLanes>(value);
#pragma unroll
            for (uint32_t mask = kLanes; mask < 32; mask *= 2) bias += __shfl_xor_sync(0xFFFFFFFFu, bias, mask);
#pragma unroll
            for (int i = 0; i < kMine; ++i) mean[i] = value[i];
        }
        at += 32 * inKey;
        most = 0;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            mean[i] += bias;
            most = max(most, (uint32_t)__double2hiint(mean[i]) & 0x7FF00000u);
        }
        most = __reduce_max_sync(0xFFFFFFFFu, most) >> 20;
        const bool broken = most == 0x7FFu;
        const int e = min(max((int)most - 1023 - 6, kLeastExponent), kMostExponent);  // (the mean is the sum / 64)
        const double down = __hiloint2double((1023 - e) << 20, 0);
        const float up = power_of_two(e - 6);
        uint32_t out[kMine / 2];
#pragma unroll
        for (int i = 0; i < kMine; i += 2) {
            float v[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) v[k] = broken ? NAN : (float)max(min(__double2int_rn(mean[i + k] * down), 127), -127) * up;
            out[i / 2] = pack_bf16x2(v[0], v[1]);
        }
        const uint32_t perPage = max(1u, pageTokens >> kBlockShift), place = (key0 & (pageTokens - 1u)) >> kBlockShift;
        if (lastPage >= a.pageCount) continue;  // (nowhere to keep it)
        uint16_t *to = a.means + (((size_t)lastPage * a.kvHeads + head) * perPage + (pageTokens > kTileKeys ? place : 0u)) * DIM + at;
        if (kMine == 8) *reinterpret_cast<uint4 *>(to) = make_uint4(out[0], out[1 % (kMine / 2)], out[2 % (kMine / 2)], out[3 % (kMine / 2)]);
        else if (kMine == 4) *reinterpret_cast<uint2 *>(to) = make_uint2(out[0], out[1 % (kMine / 2)]);
        else *reinterpret_cast<uint32_t *>(to) = out[0];
    }
}

// ---- selection -----------------------------------------------------------------------------------

// Scores: the blocks' means times the rows' queries, 16 blocks a warp at a time on mma.sync.  Both factors are whole numbers of at
// most 7 bits times a power of two of their own (the means as they are held, the queries as they are staged), so that every sum is below 2^23 of
// its unit and exact in whatever order; the largest of a row's heads is the score.  The scores wanted are found by counting them in 256 ranges
// of equal width, those of the range that holds the last one wanted in 256 ranges again, and so on until a few are left, which are compared with
// one another, or equal ones, of which the first are taken.
//
// Two forms.  k_select_split: a cluster of CTAs for each row and head, which share the blocks; the first of them gets the others' scores and
// makes the list.  k_select_rows: some neighbouring rows a CTA, which read the means of their request once; a warp makes a list.
// Bound by latency: look-up, queries, table and means, exchange, ranges, list, one after the other.  2048 blocks of 8 heads of 128 for one row 8.1 us
// (with one CTA of 512 threads a head and a search by halves 22.4; a cluster and two bits at a time 11.9).  In an instrumented copy 14.3 thousand cycles of
// the list's CTA: 1430 look-up and queries, 2970 scores, 680 exchange, 1260 for the least and the greatest score, 3750 one level of ranges, 1390 the few
// left, 2280 the list.  64 ragged requests of up to 256 blocks 8.4 us (8.0 thousand cycles); prompts of up to 613 rows, 2110 rows of 7 heads a group
// over up to 312 blocks, 18.7 (47 % of the issue slots while active).
constexpr uint32_t kRowsWarps = 8;        // of k_select_rows
constexpr uint32_t kSelectColumns = 64;   // of a CTA's product, at most
constexpr uint32_t kMostSplit = 8;        // CTAs of a cluster, at most
constexpr uint32_t kBins = 256, kFew = 32;

struct SelectArgs {
    const uint16_t *q;
    uint32_t qStride, tokens;
    const uint16_t *means;
    uint32_t pageCount;
    const uint32_t *blockTable;
    uint32_t tableStride, tableBlocks;
    const uint32_t *rowStart, *lengths;
    uint32_t requests, heads, kvHeads, pageShift;
    uint32_t blocks, first, last;
    uint32_t *ids;
    uint32_t rows, rowColumns, columns;  // of a CTA; columns of a row: the heads of its group, to a power of two or a multiple of 8 (the last head again)
    uint32_t *errorFlag;
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// scores in their order as whole numbers; a block whose mean is no number comes before all
__device__ __forceinline__ uint32_t order_of(float score) {
    const uint32_t bits = __float_as_uint(score + 0.0f);
    return score != score ? 0xFFFFFFFFu : bits ^ ((bits >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}

__host__ __device__ constexpr uint32_t select_query_stride(uint32_t dim) { return 2u * dim + 64u; }  // bytes; 64 modulo 128: no conflicts
inline uint32_t select_smem(uint32_t dim, uint32_t columns, uint32_t rows, uint32_t tableBlocks) { return columns * select_query_stride(dim) + rows * tableBlocks * 4u; }

// What a CTA knows of its rows.
struct SelectRows {
    uint32_t request[kRowsWarps], seen[kRowsWarps];  // of each row; blocks that it sees
    int exponents[kSelectColumns];                   // of a column's largest value, where a row has more than eight
};
constexpr int kNoNumber = -1000;  // the exponent of a query with a value that is not finite
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The rows' requests and the blocks that they see (s.request and s.seen are cleared, a barrier in front and behind).
__device__ __forceinline__ void select_look_up(const SelectArgs &a, SelectRows &s, uint32_t row0, uint32_t rows, uint32_t thread, uint32_t threads) {
    for (uint32_t r = thread; r < a.requests; r += threads) {
        const uint32_t begin = __ldg(a.rowStart + r), end = __ldg(a.rowStart + r + 1), length = min(__ldg(a.lengths + r), 0x7FFFFFFFu);
        if (end < begin) *a.errorFlag = kFlagRows;
        if (end <= row0 || begin >= row0 + rows || end <= begin) continue;
        for (uint32_t i = 0; i < rows; ++i) {
            const uint32_t row = row0 + i;
            if (row < begin || row >= end) continue;
            const long long position = (long long)length - (long long)(end - row);
            uint32_t seen = position < 0 ? 0u : (uint32_t)(position >> kBlockShift) + 1u;
            if (seen > a.tableBlocks) {
                seen = a.tableBlocks;
                *a.errorFlag = kFlagTableRow;
            }
            s.request[i] = r;
            s.seen[i] = seen;
        }
    }
}
// A query as it is multiplied: whole numbers of at most 7 bits at a power of two of its largest value, times one that the row's queries share.
template <int DIM>
struct Query {
    uint32_t v[DIM / 64];
    __device__ __forceinline__ void load(const uint16_t *src) {
#pragma unroll
        for (int i = 0; i < DIM / 64; ++i) v[i] = __ldg(reinterpret_cast<const uint32_t *>(src) + (threadIdx.x & 31u) + 32 * i);
    }
    __device__ __forceinline__ int exponent() const {  // of the largest value
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < DIM / 64; ++i) most = __vmaxu2(most, v[i] & 0x7FFF7FFFu);
        most = __reduce_max_sync(0xFFFFFFFFu, max(most & 0xFFFFu, most >> 16)) >> 7;
        return most == 255u ? kNoNumber : max((int)most - 127, -100);
    }
    __device__ __forceinline__ void store(uint8_t *to, int mine, int top) const {
        const int e = max(mine, top - 60);
        const float down = power_of_two(6 - e), up = power_of_two(e - top);
#pragma unroll
        for (int i = 0; i < DIM / 64; ++i) {
            const uint32_t w = mine == kNoNumber ? 0u : v[i];  // (counts as zeros)
            const float x = fminf(fmaxf(rintf(low16(w) * down), -127.0f), 127.0f) * up, y = fminf(fmaxf(rintf(high16(w) * down), -127.0f), 127.0f) * up;
            reinterpret_cast<uint32_t *>(to)[(threadIdx.x & 31u) + 32 * i] = pack_bf16x2(x, y);
        }
    }
};
// Where column c of a row stands among the CTA's: a tile of eight holds 8 / RT columns of each of RT rows, so that what a lane gets of a row's
// tiles are columns of one row (RT 4; RT 8: of two) and the largest of them is found without a look at other lanes.
template <int RT>
__device__ __forceinline__ uint32_t column_place(uint32_t row, uint32_t c, uint32_t rowColumns) {
    constexpr uint32_t kEach = 8 / RT;
    return (row / RT * (rowColumns / kEach) + c / kEach) * 8 + row % RT * kEach + c % kEach;
}
// a row's columns, up to eight, by one warp
template <int DIM, int RT, int COLUMNS>
__device__ __forceinline__ void select_stage(const SelectArgs &a, uint32_t row0, uint32_t row, uint32_t head, uint8_t *to) {
    const uint32_t group = a.heads / a.kvHeads;
    const uint16_t *src = a.q + (size_t)(row0 + row) * a.qStride + (size_t)head * group * DIM;
    Query<DIM> q[COLUMNS];
    int exponent[COLUMNS], top = -100;
#pragma unroll
    for (int c = 0; c < COLUMNS; ++c) q[c].load(src + min((uint32_t)c, group - 1u) * DIM);
#pragma unroll
    for (int c = 0; c < COLUMNS; ++c) top = max(top, exponent[c] = q[c].exponent());
#pragma unroll
    for (int c = 0; c < COLUMNS; ++c) q[c].store(to + column_place<RT>(row, c, COLUMNS) * select_query_stride(DIM), exponent[c], top);
}
// any number, by all warps, with a barrier between
template <int DIM, int RT>
__device__ __forceinline__ void select_stage_wide(const SelectArgs &a, SelectRows &s, uint32_t row0, uint32_t rows, uint32_t head, uint8_t *to, uint32_t warps) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, group = a.heads / a.kvHeads, columns = rows * a.rowColumns;
    auto column = [&](uint32_t c) { return a.q + (size_t)(row0 + c / a.rowColumns) * a.qStride + (size_t)(head * group + min(c % a.rowColumns, group - 1u)) * DIM; };
    Query<DIM> q;
    for (uint32_t c = warp; c < columns; c += warps) {
        q.load(column(c));
        const int e = q.exponent();
        if (lane == 0) s.exponents[c] = e;
    }
    __syncthreads();
    for (uint32_t c = warp; c < columns; c += warps) {
        q.load(column(c));
        int top = -100;
        for (uint32_t k = lane; k < a.rowColumns; k += 32) top = max(top, s.exponents[c / a.rowColumns * a.rowColumns + k]);
        q.store(to + column_place<RT>(c / a.rowColumns, c % a.rowColumns, a.rowColumns) * select_query_stride(DIM), s.exponents[c], __reduce_max_sync(0xFFFFFFFFu, top));
    }
}
// Scores of request r's blocks below `end`, in whole numbers of their order, to scores[row of the CTA * stride + block] for rows i0 .. i1 - 1
// (REMOTE: in another CTA's shared memory): sixteen at a time from 16 tile on, 16 step apart.  TILES: of eight columns for RT rows, 0 for any number.
template <int DIM, int RT, int TILES, bool REMOTE>
__device__ __forceinline__ void select_score(const SelectArgs &a, const uint8_t *queries, uint32_t head, uint32_t r, uint32_t end, uint32_t tile, uint32_t step, uint32_t i0, uint32_t i1,
                                             uint32_t scores, uint32_t stride) {
    constexpr uint32_t kChunks = DIM / 32;
    const uint32_t lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u, perPage = max(1u, (1u << a.pageShift) >> kBlockShift), tiles = TILES ? TILES : a.rowColumns * RT / 8;
    auto page_of = [&](uint32_t base) {  // of the mean of block base + lane % 16
        const uint32_t b = base + (lane & 15u);
        return b < end ? __ldg(a.blockTable + (size_t)r * a.tableStride + (((b << kBlockShift) + kTileKeys - 1u) >> a.pageShift)) : 0u;
    };
    uint32_t pageNext = page_of(16 * tile);
    for (uint32_t base = 16 * tile; base < end; base += 16 * step) {
        const uint32_t page = pageNext;
        const bool outside = page >= a.pageCount;
        uint4 v[2][kChunks];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t b = base + g + 8 * h, mine = __shfl_sync(0xFFFFFFFFu, outside ? 0u : page, g + 8 * h);
            const uint4 *src = reinterpret_cast<const uint4 *>(a.means + (((size_t)mine * a.kvHeads + head) * perPage + (b & (perPage - 1u))) * DIM) + t;
#pragma unroll
            for (uint32_t c = 0; c < kChunks; ++c) v[h][c] = a.pageCount ? __ldg(src + 4 * c) : make_uint4(0u, 0u, 0u, 0u);
        }
        pageNext = page_of(base + 16 * step);
        const uint32_t gone = __ballot_sync(0xFFFFFFFFu, outside);
        if (gone && lane == 0) *a.errorFlag = kFlagPage;
        for (uint32_t i = i0 / RT * RT; i < i1; i += RT) {
            const uint8_t *from = queries + (i / RT * tiles * 8 + g) * select_query_stride(DIM) + 16 * t;
            float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // [block g: column 2 t, 2 t + 1; block g + 8: likewise]
#pragma unroll
            for (uint32_t n = 0; n < tiles; ++n) {
                float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (uint32_t c = 0; c < kChunks; ++c) {
                    const uint4 b = *reinterpret_cast<const uint4 *>(from + n * 8 * select_query_stride(DIM) + 64 * c);
                    mma_bf16(acc, v[0][c].x, v[1][c].x, v[0][c].y, v[1][c].y, b.x, b.y);
                    mma_bf16(acc, v[0][c].z, v[1][c].z, v[0][c].w, v[1][c].w, b.z, b.w);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) best[k] = max_nan(best[k], acc[k]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t b = base + g + 8 * h;
                const bool none = gone >> (g + 8 * h) & 1u;
                auto put = [&](uint32_t row, float x) {
                    const uint32_t order = none ? 0u : order_of(x);
                    if (b >= end || row < i0 || row >= i1) return;
                    if (REMOTE) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(scores + 4 * (row * stride + b)), "r"(order) : "memory");
                    else asm volatile("st.shared.u32 [%0], %1;" ::"r"(scores + 4 * (row * stride + b)), "r"(order) : "memory");
                };
                if (RT == 8) {
                    put(i + 2 * t, best[2 * h]);
                    put(i + 2 * t + 1, best[2 * h + 1]);
                } else {
                    float x = max_nan(best[2 * h], best[2 * h + 1]);
                    if (RT == 1) {
                        x = max_nan(x, __shfl_xor_sync(0xFFFFFFFFu, x, 1));
                        x = max_nan(x, __shfl_xor_sync(0xFFFFFFFFu, x, 2));
                    }
                    if (RT == 4 || t == 0) put(i + (RT == 4 ? t : 0u), x);
                }
            }
        }
    }
}

// The `wanted` largest of n scores (more than wanted), of equal ones the first, by WARPS warps: ids first + place, ascending, to out.
struct SelectCounts {
    __align__(16) uint32_t bins[2][kBins];  // of this level, of the next
    uint2 few[kFew];          // score, place
    uint32_t least[2][16], most[2][16], above[16], same[16], held;  // of each warp
};
template <int WARPS>
__device__ __forceinline__ void select_meet() {
    if (WARPS == 1) __syncwarp();
    else __syncthreads();
}
__device__ __forceinline__ float score_of(uint32_t order) { return __uint_as_float(order ^ ((order >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }
template <int WARPS>
__device__ __forceinline__ void select_largest(const uint32_t *scores, uint32_t n, uint32_t wanted, uint32_t first, uint32_t *out, SelectCounts &s) {
    const uint32_t lane = threadIdx.x & 31u, warp = WARPS == 1 ? 0u : threadIdx.x >> 5, thread = WARPS == 1 ? lane : threadIdx.x;
    const uint32_t each = (n + 32 * WARPS - 1) / (32 * WARPS) * 32u, k0 = min(warp * each, n), k1 = min(k0 + each, n);  // a warp's run of them
    // Of the scores from `low` to `high`, which are the least and the greatest of them, `left` are wanted; those above are, those below are not.
    uint32_t low = 0xFFFFFFFFu, high = 0u, left = wanted, few = n;
    auto all_warps = [&](uint32_t *lows, uint32_t *highs) {
        low = __reduce_min_sync(0xFFFFFFFFu, low), high = __reduce_max_sync(0xFFFFFFFFu, high);
        if (WARPS > 1 && lane == 0) lows[warp] = low, highs[warp] = high;
        select_meet<WARPS>();
        if (WARPS > 1) low = __reduce_min_sync(0xFFFFFFFFu, lows[lane % WARPS]), high = __reduce_max_sync(0xFFFFFFFFu, highs[lane % WARPS]);
    };
    for (uint32_t k = thread; k < kBins; k += 32 * WARPS) s.bins[0][k] = 0u;
    if (thread == 0) s.held = 0u;
#pragma unroll 4
    for (uint32_t k = k0 + lane; k < k1; k += 32) low = min(low, scores[k]), high = max(high, scores[k]);
    all_warps(s.least[1], s.most[1]);
    for (uint32_t level = 0; low != high && few > kFew; ++level) {
        // Ranges of equal width, twice of the scores' values (which lie evenly), then of the whole numbers that stand for them (which ends).
        // Scores that are no number, or of no mean, are the last and the first of these.
        const uint32_t least = low, most = high, *bins = s.bins[level & 1u];
        const bool values = level < 2 && least > 0x00800000u && most < 0xFF800000u;
        const float from = score_of(least), widthInverse = (kBins - 1) / (score_of(most) - from);
        const uint32_t shift = max(0, 24 - __clz(most - least));
        auto bin_of = [&](uint32_t v) { return values ? min((uint32_t)((score_of(v) - from) * widthInverse), kBins - 1u) : (v - least) >> shift; };
#pragma unroll 4
        for (uint32_t k = k0 + lane; k < k1; k += 32) {
            const uint32_t v = scores[k];
            if (v >= least && v <= most) atomicAdd(&s.bins[level & 1u][bin_of(v)], 1u);
        }
        select_meet<WARPS>();
        // the range that holds the last one wanted: a lane has eight, the uppermost lane the last
        uint32_t counts[kBins / 32], sum = 0;
#pragma unroll
        for (uint32_t i = 0; i < kBins / 32; i += 4) {
            const uint4 four = *reinterpret_cast<const uint4 *>(bins + lane * (kBins / 32) + i);
            counts[i] = four.x, counts[i + 1] = four.y, counts[i + 2] = four.z, counts[i + 3] = four.w;
            sum += four.x + four.y + four.z + four.w;
        }
        for (uint32_t k = thread; k < kBins; k += 32 * WARPS) s.bins[~level & 1u][k] = 0u;
        uint32_t above = sum;  // in this lane's ranges and above
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t v = __shfl_down_sync(0xFFFFFFFFu, above, d);
            if (lane + d < 32) above += v;
        }
        above -= sum;
        const bool here = above < left && above + sum >= left;
        uint32_t bin = 0, over = above, inside = 0;
        bool found = false;
#pragma unroll
        for (int i = kBins / 32 - 1; i >= 0; --i)
            if (!found) {
                if (over + counts[i] >= left) bin = lane * (kBins / 32) + i, inside = counts[i], found = true;
                else over += counts[i];
            }
        const uint32_t source = 31u - __clz(__ballot_sync(0xFFFFFFFFu, here));
        bin = __shfl_sync(0xFFFFFFFFu, bin, source), few = __shfl_sync(0xFFFFFFFFu, inside, source), left -= __shfl_sync(0xFFFFFFFFu, over, source);
        low = 0xFFFFFFFFu, high = 0u;
#pragma unroll 4
        for (uint32_t k = k0 + lane; k < k1; k += 32) {
            const uint32_t v = scores[k];
            if (v >= least && v <= most && bin_of(v) == bin) low = min(low, v), high = max(high, v);
        }
        all_warps(s.least[level & 1u], s.most[level & 1u]);
    }
    const bool equal = low == high;
    // a few scores: the last one wanted is the `left`-th largest of them, with its place
    uint32_t bound = low, place = 0xFFFFFFFFu;
    if (!equal) {
        for (uint32_t k = k0 + lane; k < k1; k += 32) {
            const uint32_t v = scores[k];
            if (v >= low && v <= high) s.few[atomicAdd(&s.held, 1u)] = make_uint2(v, k);
        }
        select_meet<WARPS>();
        const uint2 mine = s.few[min(lane, few - 1u)];
        uint32_t before = 0;
        for (uint32_t i = 0; i < few; ++i) {
            const uint2 other = s.few[i];
            before += other.x > mine.x || (other.x == mine.x && other.y < mine.y);
        }
        const uint32_t who = __ballot_sync(0xFFFFFFFFu, lane < few && before == left - 1u);
        bound = __shfl_sync(0xFFFFFFFFu, mine.x, __ffs(who) - 1), place = __shfl_sync(0xFFFFFFFFu, mine.y, __ffs(who) - 1);
    }
    // those above the bound, and of those at it the first (equal: `left` of them; otherwise up to the place)
    uint32_t aboveBefore = 0, sameBefore = 0;
    auto above_it = [&](uint32_t v, uint32_t k) { return v > bound || (!equal && v == bound && k <= place); };
    auto at_it = [&](uint32_t v) { return equal && v == bound; };
    if (WARPS > 1) {
        uint32_t above = 0, same = 0;
        for (uint32_t k = k0 + lane; k < k1; k += 32) {
            const uint32_t v = scores[k];
            above += above_it(v, k), same += at_it(v);
        }
        above = __reduce_add_sync(0xFFFFFFFFu, above), same = __reduce_add_sync(0xFFFFFFFFu, same);
        if (lane == 0) s.above[warp] = above, s.same[warp] = same;
        select_meet<WARPS>();
        const bool front = (int)lane < (int)warp;
        aboveBefore = __reduce_add_sync(0xFFFFFFFFu, front ? s.above[lane % WARPS] : 0u), sameBefore = __reduce_add_sync(0xFFFFFFFFu, front ? s.same[lane % WARPS] : 0u);
    }
    const uint32_t under = (1u << lane) - 1u;
    for (uint32_t k = k0; k < k1; k += 32) {
        const bool there = k + lane < k1;
        const uint32_t v = there ? scores[k + lane] : 0u;
        const bool up = there && above_it(v, k + lane), same = there && at_it(v);
        const uint32_t ups = __ballot_sync(0xFFFFFFFFu, up), sames = __ballot_sync(0xFFFFFFFFu, same);
        const uint32_t at = sameBefore + __popc(sames & under);
        if (up || (same && at < left)) out[aboveBefore + __popc(ups & under) + min(at, left)] = first + k + lane;
        aboveBefore += __popc(ups);
        sameBefore += __popc(sames);
    }
}
// What of a list needs no scores, by `threads` threads; whether that is all of it.
__device__ __forceinline__ bool select_always(const SelectArgs &a, uint32_t *out, uint32_t seen, uint32_t thread, uint32_t threads) {
    if (seen <= a.blocks) {
        for (uint32_t k = thread; k < a.blocks; k += threads) out[k] = k < seen ? k : FF_NO_SLOT;
        return true;
    }
    for (uint32_t k = thread; k < a.first; k += threads) out[k] = k;
    for (uint32_t k = thread; k < a.last; k += threads) out[a.blocks - a.last + k] = seen - a.last + k;
    return a.blocks == a.first + a.last;
}

template <int DIM, int TILES, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) k_select_split(const __grid_constant__ SelectArgs a) {
    constexpr uint32_t kWarps = WARPS;
    extern __shared__ __align__(16) uint8_t selectSmem[];
    __shared__ SelectRows s;
    __shared__ SelectCounts counts;
    const uint32_t tid = threadIdx.x, warp = tid >> 5;
    const uint32_t head = blockIdx.z, row = blockIdx.y, cta = blockIdx.x, ctas = gridDim.x;
    uint32_t *scores = reinterpret_cast<uint32_t *>(selectSmem + a.columns * select_query_stride(DIM));  // those of the cluster's first CTA count
    if (tid == 0) s.request[0] = FF_NO_SLOT, s.seen[0] = 0u;
    pdl_enter();
    if (ctas > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // (the first CTA is there to be written to: waited for below)
    __syncthreads();
    // a warp a column, where there are no more: its exponent in front of the look at the requests, the numbers behind
    [[maybe_unused]] Query<DIM> q;
    [[maybe_unused]] int exponent = kNoNumber;
    if (TILES == 1 && warp < 8) {
        q.load(a.q + (size_t)row * a.qStride + (size_t)(head * (a.heads / a.kvHeads) + min(warp, a.heads / a.kvHeads - 1u)) * DIM);
        exponent = q.exponent();
        if ((tid & 31u) == 0) s.exponents[warp] = exponent;
    }
    if (TILES != 1) select_stage_wide<DIM, 1>(a, s, row, 1, head, selectSmem, kWarps);
    select_look_up(a, s, row, 1, (tid + 32 * (kWarps - 8)) % (32 * kWarps), 32 * kWarps);  // (from the ninth warp on, where there is one)
    __syncthreads();
    if (TILES == 1) {
        if (warp < 8) {
            int top = -100;
#pragma unroll
            for (int c = 0; c < 8; ++c) top = max(top, s.exponents[c]);
            q.store(selectSmem + warp * select_query_stride(DIM), exponent, top);
        }
        __syncthreads();
    }
    if (ctas > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    const uint32_t seen = s.seen[0], wanted = a.blocks - a.first - a.last;
    if (seen > a.blocks && wanted) {
        const uint32_t tile = cta * kWarps + warp, step = ctas * kWarps;
        if (cta) select_score<DIM, 1, TILES, true>(a, selectSmem, head, s.request[0], seen - a.last, tile, step, 0, 1, map_to_cta(sm_addr(scores), 0), 0);
        else select_score<DIM, 1, TILES, false>(a, selectSmem, head, s.request[0], seen - a.last, tile, step, 0, 1, sm_addr(scores), 0);
    }
    if (ctas > 1) cluster_sync_all();
    else __syncthreads();
    if (cta) return;
    uint32_t *out = a.ids + ((size_t)row * a.kvHeads + head) * a.blocks;
    if (select_always(a, out, seen, tid, 32 * kWarps)) return;
    select_largest<kWarps>(scores + a.first, seen - a.last - a.first, wanted, a.first, out + a.first, counts);
}

template <int DIM, int RT, int TILES>
__global__ void __launch_bounds__(32 * kRowsWarps, DIM == 256 ? 2 : DIM == 128 ? 3 : 4) k_select_rows(const __grid_constant__ SelectArgs a) {
    extern __shared__ __align__(16) uint8_t selectSmem[];
    __shared__ SelectRows s;
    __shared__ SelectCounts counts[kRowsWarps];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const uint32_t head = blockIdx.y, row0 = blockIdx.x * a.rows, rows = min(a.rows, a.tokens - row0);
    uint32_t *scores = reinterpret_cast<uint32_t *>(selectSmem + a.columns * select_query_stride(DIM));  // [rows][tableBlocks]
    if (tid < kRowsWarps) s.request[tid] = FF_NO_SLOT, s.seen[tid] = 0u;
    pdl_enter();
    __syncthreads();
    const uint32_t wanted = a.blocks - a.first - a.last;
    if (TILES == 0) select_stage_wide<DIM, RT>(a, s, row0, rows, head, selectSmem, kRowsWarps);
    else if (warp < rows) select_stage<DIM, RT, (TILES ? TILES : 1) * 8 / RT>(a, row0, warp, head, selectSmem);
    select_look_up(a, s, row0, rows, tid, 32 * kRowsWarps);
    __syncthreads();
    for (uint32_t i0 = 0, i1; i0 < rows; i0 = i1) {  // request by request
        uint32_t end = 0;  // blocks that a row of the request may choose
        for (i1 = i0; i1 < rows && s.request[i1] == s.request[i0]; ++i1)
            if (s.seen[i1] > a.blocks) end = max(end, s.seen[i1] - a.last);
        if (s.request[i0] == FF_NO_SLOT || !wanted) continue;
        select_score<DIM, RT, TILES, false>(a, selectSmem, head, s.request[i0], end, warp, kRowsWarps, i0, i1, sm_addr(scores), a.tableBlocks);
    }
    __syncthreads();
    if (warp >= rows) return;
    const uint32_t seen = s.seen[warp];
    uint32_t *out = a.ids + ((size_t)(row0 + warp) * a.kvHeads + head) * a.blocks;
    if (select_always(a, out, seen, lane, 32)) return;
    select_largest<1>(scores + warp * a.tableBlocks + a.first, seen - a.last - a.first, wanted, a.first, out + a.first, counts[warp]);
}

KernelSmemMemo meansMemo[3], splitMemo[3][4], rowsMemo[3][6];

}  // namespace

bool launch_block_means(FFAttention *att, const uint8_t *pages, uint32_t pageCount, const uint32_t *blockTable, uint32_t tableStride, uint32_t tableKeys,
                        const uint32_t *oldLengths, const uint32_t *newLengths, uint32_t requests, uint16_t *means, cudaStream_t stream, const char **error) {
    const FFAttentionConfig &c = att->cfg;
    const MeansArgs args{pages, pageCount, blockTable, tableStride, tableKeys, oldLengths, newLengths, requests, c.kvHeads, (uint32_t)__builtin_ctz(c.pageTokens),
                         page_layout(c), means, att->errorFlag};
    const uint64_t most = ((uint64_t)requests * (tableKeys / kTileKeys) * c.kvHeads + kMeansThreads / 32 - 1) / (kMeansThreads / 32);
    const uint32_t grid = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(most, (uint32_t)att->smCount)), smem = kMeansThreads / 32 * means_bytes(c.headDim);
    auto launch = [&](auto kernel, KernelSmemMemo &memo) {
        if (!memo.prepare(kernel, att->device, smem, kMeansThreads, nullptr, error)) return false;
        return launched(att, launch_pdl(kernel, dim3(grid), dim3(kMeansThreads), smem, stream, args), "k_block_means", error);
    };
    return c.headDim == 256 ? launch(k_block_means<256>, meansMemo[2]) : c.headDim == 128 ? launch(k_block_means<128>, meansMemo[1]) : launch(k_block_means<64>, meansMemo[0]);
}

bool launch_select_blocks(FFAttention *att, const uint16_t *q, uint32_t qStride, uint32_t tokens, const uint16_t *means, uint32_t pageCount,
                          const uint32_t *blockTable, uint32_t tableStride, uint32_t tableBlocks, const uint32_t *rowStart, const uint32_t *lengths,
                          uint32_t requests, uint32_t blocks, uint32_t first, uint32_t last, uint32_t *ids, cudaStream_t stream, const char **error) {
    const FFAttentionConfig &c = att->cfg;
    const uint32_t group = c.heads / c.kvHeads, sms = (uint32_t)att->smCount;
    SelectArgs args{q, qStride, tokens, means, pageCount, blockTable, tableStride, tableBlocks, rowStart, lengths, requests, c.heads, c.kvHeads,
                    (uint32_t)__builtin_ctz(c.pageTokens), blocks, first, last, ids, 1, (group + 7u) & ~7u, 0, att->errorFlag};
    const uint64_t lists = (uint64_t)tokens * c.kvHeads;
    const int dim = c.headDim == 256 ? 2 : c.headDim == 128 ? 1 : 0;
    auto of_dim = [&](auto launch) {  // launch(values of a head, as a constant)
        return dim == 2 ? launch(std::integral_constant<int, 256>()) : dim == 1 ? launch(std::integral_constant<int, 128>()) : launch(std::integral_constant<int, 64>());
    };
    // A cluster a list where lists are few, or most rows another request's: these have no means in common (100 requests of 8 heads of 512
    // blocks 33 us, eight rows a CTA 68; one request's 300 rows of 8 heads of 312 blocks 27 us eight a CTA).
    if (lists <= 4ull * sms || ((uint64_t)tokens < 4ull * requests && tokens <= 65535)) {
        // Sixteen warps where a CTA has an SM for itself (at 256 values a head their registers leave room for eight); CTAs to fill
        // the GPU, as long as each of them has its warps' blocks.
        const uint32_t warps = lists <= sms && dim < 2 ? 16u : 8u;
        uint32_t ctas = 1;
        while (ctas < kMostSplit && 2 * ctas * lists <= (warps == 16 ? sms : 2 * sms) && 2 * ctas * warps * 16 <= tableBlocks) ctas *= 2;
        args.columns = args.rowColumns;
        const uint32_t smem = select_smem(c.headDim, args.columns, 1, tableBlocks);
        auto launch = [&](auto kernel, KernelSmemMemo &memo) {
            if (!memo.prepare(kernel, att->device, smem, 32 * warps, nullptr, error)) return false;
            cudaLaunchConfig_t config{};
            config.gridDim = dim3(ctas, tokens, c.kvHeads);
            config.blockDim = dim3(32 * warps);
            config.dynamicSmemBytes = smem;
            config.stream = stream;
            cudaLaunchAttribute attributes[2]{};
            attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attributes[0].val.programmaticStreamSerializationAllowed = 1;
            attributes[1].id = cudaLaunchAttributeClusterDimension;
            attributes[1].val.clusterDim.x = ctas;
            attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
            config.attrs = attributes;
            config.numAttrs = 2;
            return launched(att, cudaLaunchKernelEx(&config, kernel, args), "k_select_split", error);
        };
        return of_dim([&](auto d) {
            constexpr int kMost = d.value == 256 ? 8 : 16;
            const bool one = args.rowColumns == 8;
            if (warps == 16) return one ? launch(k_select_split<d.value, 1, kMost>, splitMemo[dim][0]) : launch(k_select_split<d.value, 0, kMost>, splitMemo[dim][1]);
            return one ? launch(k_select_split<d.value, 1, 8>, splitMemo[dim][2]) : launch(k_select_split<d.value, 0, 8>, splitMemo[dim][3]);
        });
    }
    // A warp's list each, as far as the columns and the shared memory for their scores go.
    uint32_t narrow = group > 8 ? args.rowColumns : 1u;
    while (narrow < group) narrow *= 2;
    args.rows = std::min(kRowsWarps, kSelectColumns / narrow);
    while (args.rows > 1 && select_smem(c.headDim, std::max(8u, args.rows * narrow), args.rows, tableBlocks) > 100u * 1024u) args.rows /= 2;
    const uint32_t together = args.rows < 4 ? 1u : narrow == 1 && args.rows == 8 ? 8u : 4u;  // rows of a tile of columns
    if (together > 1) args.rowColumns = std::max(narrow, 8u / together);
    args.rows = args.rows / together * together;
    args.columns = args.rows * args.rowColumns;
    const uint32_t smem = select_smem(c.headDim, args.columns, args.rows, tableBlocks), tiles = args.rowColumns * together / 8;
    auto launch = [&](auto kernel, KernelSmemMemo &memo) {
        if (!memo.prepare(kernel, att->device, smem, 32 * kRowsWarps, nullptr, error)) return false;
        return launched(att, launch_pdl(kernel, dim3((tokens + args.rows - 1) / args.rows, c.kvHeads), dim3(32 * kRowsWarps), smem, stream, args), "k_select_rows", error);
    };
    return of_dim([&](auto d) {
        if (together == 8) return launch(k_select_rows<d.value, 8, 1>, rowsMemo[dim][0]);
        if (together == 1) return launch(k_select_rows<d.value, 1, 0>, rowsMemo[dim][1]);
        return tiles == 1 ? launch(k_select_rows<d.value, 4, 1>, rowsMemo[dim][2]) : tiles == 2 ? launch(k_select_rows<d.value, 4, 2>, rowsMemo[dim][3])
             : tiles == 4 ? launch(k_select_rows<d.value, 4, 4>, rowsMemo[dim][4]) : launch(k_select_rows<d.value, 4, 0>, rowsMemo[dim][5]);
    });
}

}  // namespace ff

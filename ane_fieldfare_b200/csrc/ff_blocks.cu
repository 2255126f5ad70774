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

// A warp takes a block of a key/value head: 64 keys of code * scale + bias summed in 64 bits, where the sum is exact unless the
// scales of a block are 2^35 apart; then whole numbers of 2^(e - 6), e the exponent of the largest value: 7 bits and a sign, which
// bf16 holds.  So nothing about a mean depends on the order of sums.
constexpr int kMeansThreads = 256;

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

template <int DIM>
__global__ void __launch_bounds__(kMeansThreads) k_block_means(const __grid_constant__ MeansArgs a) {
    constexpr uint32_t CB = DIM / 2, NG = DIM / 64, kLanes = CB / 8, kKeys = 32 / kLanes;  // lanes a key, keys at once
    constexpr int kRounds = kKeys == 8 ? 3 : kKeys == 4 ? 2 : 1, kMine = 16 >> kRounds;
    __shared__ uint32_t first[kMeansThreads + 1], warpSums[kMeansThreads / 32];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
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
    const unsigned long long items = (unsigned long long)total * a.kvHeads;
    for (unsigned long long item = (unsigned long long)blockIdx.x * (kMeansThreads / 32) + warp; item < items; item += (unsigned long long)gridDim.x * (kMeansThreads / 32)) {
        uint32_t n = (uint32_t)(item / a.kvHeads);
        const uint32_t head = (uint32_t)(item % a.kvHeads);
        uint32_t low = 0, high = kMeansThreads;
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
        const uint32_t key0 = (s.begin + n) << kBlockShift;
        // a lane holds the page of one piece of the block
        const uint32_t pieces = kTileKeys >> pieceShift;
        uint32_t page = 0;
        if (lane < pieces) page = __ldg(a.blockTable + (size_t)r * a.tableStride + ((key0 + (lane << pieceShift)) >> a.pageShift));
        const bool hole = __any_sync(0xFFFFFFFFu, page >= a.pageCount);
        const uint32_t lastPage = __shfl_sync(0xFFFFFFFFu, page, pieces - 1u);
        if (hole && lane == 0) *a.errorFlag = kFlagPage;
        if (lastPage >= a.pageCount) continue;
        double value[16], bias = 0.0;
#pragma unroll
        for (int i = 0; i < 16; ++i) value[i] = 0.0;
        if (!hole) {
#pragma unroll 4
            for (uint32_t k = 0; k < kTileKeys / kKeys; ++k) {
                const uint32_t key = k * kKeys + keyLane;
                const uint32_t at = (key0 + key) & (pageTokens - 1u);
                const uint8_t *block = a.pages + ((size_t)__shfl_sync(0xFFFFFFFFu, page, key >> pieceShift) * a.kvHeads + head) * a.page.blockBytes;
                const uint2 codes = __ldg(reinterpret_cast<const uint2 *>(block + (size_t)at * CB + inKey * 8));
                const uint32_t word = __ldg(reinterpret_cast<const uint32_t *>(block + a.page.keyWords + (size_t)at * (NG * 4)) + inKey / (kLanes / NG));
                const double scale = (double)low16(word);
                bias += (double)high16(word);
#pragma unroll
                for (int i = 0; i < 16; ++i)  // (2^52 + code less 2^52: a conversion takes longer)
                    value[i] = fma(scale, __hiloint2double(0x43300000, (int)((i < 8 ? codes.x : codes.y) >> (4 * (i & 7)) & 15u)) - 0x1p52, value[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) value[i] += bias;
        // the keys' lanes joined: each round a lane gives half of its values and takes the other half's of its partner
        uint32_t at = 16 * inKey;
#pragma unroll
        for (int round = 0; round < kRounds; ++round) {
            const int half = 8 >> round;
            const uint32_t mask = kLanes << round;
            const bool upper = lane & mask;
            if (upper) at += half;
#pragma unroll
            for (int i = 0; i < half; ++i) {
                const double give = upper ? value[i] : value[i + half], keep = upper ? value[i + half] : value[i];
                value[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, mask);
            }
        }
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < kMine; ++i) most = max(most, (uint32_t)__double2hiint(value[i]) & 0x7FF00000u);
        most = __reduce_max_sync(0xFFFFFFFFu, most) >> 20;
        const bool broken = most == 0x7FFu;
        const int e = min(max((int)most - 1023 - 6, kLeastExponent), kMostExponent);  // (the mean is the sum / 64)
        const double down = __hiloint2double((1023 - e) << 20, 0);
        const float up = power_of_two(e - 6);
        uint32_t out[(kMine + 1) / 2];
#pragma unroll
        for (int i = 0; i < kMine; i += 2) {
            float v[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) v[k] = broken ? NAN : (float)fmin(fmax(rint(value[i + k] * down), -127.0), 127.0) * up;
            out[i / 2] = pack_bf16x2(v[0], v[1]);
        }
        const uint32_t perPage = max(1u, pageTokens >> kBlockShift), place = (key0 & (pageTokens - 1u)) >> kBlockShift;
        uint16_t *to = a.means + (((size_t)lastPage * a.kvHeads + head) * perPage + (pageTokens > kTileKeys ? place : 0u)) * DIM + at;
        if (kMine == 8) *reinterpret_cast<uint4 *>(to) = make_uint4(out[0], out[1 % ((kMine + 1) / 2)], out[2 % ((kMine + 1) / 2)], out[3 % ((kMine + 1) / 2)]);
        else if (kMine == 4) *reinterpret_cast<uint2 *>(to) = make_uint2(out[0], out[1 % ((kMine + 1) / 2)]);
        else *reinterpret_cast<uint32_t *>(to) = out[0];
    }
}

// ---- selection -----------------------------------------------------------------------------------

// A CTA takes `rows` neighbouring rows of one key/value head.  Scores: the blocks' means times the rows' queries, 16 blocks a
// warp at a time on mma.sync.  Both factors are whole numbers of at most 7 bits times a power of two of their own (the means as they are
// held, the queries as they are staged), so that every sum is below 2^23 of its unit and exact in whatever order; the largest of a
// row's heads is the score.  Then the bound that as many scores reach as are wanted, by halving the range of scores as whole
// numbers, until the number that reaches it is the number wanted or the range is one score, of which the first blocks are taken.
constexpr int kSelectThreads = 512, kSelectWarps = kSelectThreads / 32;
constexpr uint32_t kSelectRows = 8;  // rows of a CTA, at most: the columns of a product

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
    uint32_t rows, rowColumns;  // of a CTA; columns of a row: the heads of its group, to a power of two or a multiple of 8
    uint32_t *errorFlag;
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
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

template <int DIM>
__global__ void __launch_bounds__(kSelectThreads) k_select_blocks(const __grid_constant__ SelectArgs a) {
    constexpr uint32_t kStride = select_query_stride(DIM), kChunks = DIM / 32;
    extern __shared__ __align__(16) uint8_t selectSmem[];
    __shared__ int exponents[64];
    __shared__ uint32_t requestOf[kSelectRows], seenBlocks[kSelectRows], counts[2][kSelectWarps], greater[kSelectWarps], equal[kSelectWarps];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, g = lane >> 2, t = lane & 3u;
    const uint32_t head = blockIdx.y, row0 = blockIdx.x * a.rows, rows = min(a.rows, a.tokens - row0), group = a.heads / a.kvHeads;
    const uint32_t columns = (a.rows * a.rowColumns + 7u) & ~7u;
    uint32_t *scores = reinterpret_cast<uint32_t *>(selectSmem + columns * kStride);  // [rows][tableBlocks]
    if (tid < kSelectRows) requestOf[tid] = FF_NO_SLOT, seenBlocks[tid] = 0u;
    pdl_enter();
    __syncthreads();

    // ---- the rows' requests and the blocks that they see ----
    for (uint32_t r = tid; r < a.requests; r += kSelectThreads) {
        const uint32_t begin = __ldg(a.rowStart + r), end = __ldg(a.rowStart + r + 1);
        if (end < begin && blockIdx.x == 0) *a.errorFlag = kFlagRows;
        if (end <= row0 || begin >= row0 + rows || end <= begin) continue;
        const uint32_t length = min(__ldg(a.lengths + r), 0x7FFFFFFFu);
        for (uint32_t i = 0; i < rows; ++i) {
            const uint32_t row = row0 + i;
            if (row < begin || row >= end) continue;
            const long long position = (long long)length - (long long)(end - row);
            uint32_t seen = position < 0 ? 0u : (uint32_t)(position >> kBlockShift) + 1u;
            if (seen > a.tableBlocks) {
                seen = a.tableBlocks;
                *a.errorFlag = kFlagTableRow;
            }
            requestOf[i] = r;
            seenBlocks[i] = seen;
        }
    }
    __syncthreads();
    const uint32_t wanted = a.blocks - a.first - a.last;
    bool any = false;  // whether some row has more blocks than it takes
#pragma unroll 1
    for (uint32_t i = 0; i < rows; ++i) any |= seenBlocks[i] > a.blocks;

    if (any && wanted) {
        // ---- queries: whole numbers of at most 7 bits, at a power of two of the head's largest value ----
        // (exponent of a column's largest value, then of its row's largest)
        for (uint32_t c = warp; c < columns; c += kSelectWarps) {
            const uint32_t i = c / a.rowColumns, h = min(c % a.rowColumns, group - 1u);
            uint32_t most = 0;
            if (i < rows) {
                const uint16_t *src = a.q + (size_t)(row0 + i) * a.qStride + (head * group + h) * DIM;
#pragma unroll
                for (uint32_t d = 2 * lane; d < DIM; d += 64) most = __vmaxu2(most, __ldg(reinterpret_cast<const uint32_t *>(src + d)) & 0x7FFF7FFFu);
            }
            most = __reduce_max_sync(0xFFFFFFFFu, max(most & 0xFFFFu, most >> 16)) >> 7;
            if (lane == 0 && c % a.rowColumns < 64u) exponents[c % 64u] = most == 255u ? -1000 : max((int)most - 127, -100);
        }
        __syncthreads();
        for (uint32_t c = warp; c < columns; c += kSelectWarps) {
            const uint32_t i = c / a.rowColumns, h = min(c % a.rowColumns, group - 1u);
            int top = -100;
            for (uint32_t k = 0; k < a.rowColumns; ++k) top = max(top, exponents[(i * a.rowColumns + k) % 64u]);
            const int mine = exponents[c % 64u];
            const bool none = i >= rows || mine == -1000;  // (a head with a value that is no number counts as zeros)
            const int e = max(mine, top - 60);
            const float down = power_of_two(6 - e), up = power_of_two(e - top);
            const uint16_t *src = a.q + (size_t)(row0 + (none ? 0u : i)) * a.qStride + (head * group + h) * DIM;
#pragma unroll
            for (uint32_t d = 2 * lane; d < DIM; d += 64) {
                const uint32_t v = none ? 0u : __ldg(reinterpret_cast<const uint32_t *>(src + d));
                const float x = fminf(fmaxf(rintf(low16(v) * down), -127.0f), 127.0f) * up, y = fminf(fmaxf(rintf(high16(v) * down), -127.0f), 127.0f) * up;
                *reinterpret_cast<uint32_t *>(selectSmem + c * kStride + 2 * d) = pack_bf16x2(x, y);
            }
        }
        __syncthreads();

        // ---- scores, request by request ----
        const uint32_t perPage = max(1u, (1u << a.pageShift) >> kBlockShift);
        for (uint32_t i0 = 0, i1; i0 < rows; i0 = i1) {
            uint32_t end = 0;  // blocks that a row of the request may choose
            for (i1 = i0; i1 < rows && requestOf[i1] == requestOf[i0]; ++i1)
                if (seenBlocks[i1] > a.blocks) end = max(end, seenBlocks[i1] - a.last);
            const uint32_t r = requestOf[i0];
            if (r == FF_NO_SLOT || end == 0) continue;
            auto page_of = [&](uint32_t base) {  // of the mean of block base + lane, lane < 16
                const uint32_t b = base + (lane & 15u);
                return b < end ? __ldg(a.blockTable + (size_t)r * a.tableStride + (((b << kBlockShift) + kTileKeys - 1u) >> a.pageShift)) : FF_NO_PAGE;
            };
            uint32_t pageNext = page_of(16 * warp);
            for (uint32_t base = 16 * warp; base < end; base += 16 * kSelectWarps) {
                const uint32_t page = pageNext;
                uint4 v[2][kChunks];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t b = base + g + 8 * h, mine = __shfl_sync(0xFFFFFFFFu, page, g + 8 * h);
                    const uint16_t *src = a.means + (((size_t)mine * a.kvHeads + head) * perPage + (b & (perPage - 1u))) * DIM + 8 * t;
#pragma unroll
                    for (uint32_t c = 0; c < kChunks; ++c) v[h][c] = mine < a.pageCount ? __ldg(reinterpret_cast<const uint4 *>(src + 32 * c)) : make_uint4(0u, 0u, 0u, 0u);
                }
                pageNext = page_of(base + 16 * kSelectWarps);
                float best[2][2] = {{-INFINITY, -INFINITY}, {-INFINITY, -INFINITY}};  // [block g, g + 8][column 2 t, 2 t + 1]
                for (uint32_t n = 0; n < columns; n += 8) {
                    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (uint32_t c = 0; c < kChunks; ++c) {
                        const uint4 b = *reinterpret_cast<const uint4 *>(selectSmem + (n + g) * kStride + 64 * c + 16 * t);
                        mma_bf16(acc, v[0][c].x, v[1][c].x, v[0][c].y, v[1][c].y, b.x, b.y);
                        mma_bf16(acc, v[0][c].z, v[1][c].z, v[0][c].w, v[1][c].w, b.z, b.w);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        // (a NaN mean makes all columns NaN: it stays)
                        best[k >> 1][k & 1] = acc[k] != acc[k] ? acc[k] : fmaxf(best[k >> 1][k & 1], acc[k]);
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t k0 = order_of(best[h][0]), k1 = order_of(best[h][1]);
                    if (__shfl_sync(0xFFFFFFFFu, page, g + 8 * h) >= a.pageCount) k0 = k1 = 0u;
                    const uint32_t b = base + g + 8 * h;
                    if (a.rowColumns > 1) k0 = k1 = max(k0, k1);
                    if (a.rowColumns > 2) k0 = max(k0, __shfl_xor_sync(0xFFFFFFFFu, k0, 1));
                    if (a.rowColumns > 4) k0 = max(k0, __shfl_xor_sync(0xFFFFFFFFu, k0, 2));
                    if (b >= end) continue;
                    if (a.rowColumns == 1) {
                        if (2 * t >= i0 && 2 * t < i1) scores[2 * t * a.tableBlocks + b] = k0;
                        if (2 * t + 1 >= i0 && 2 * t + 1 < i1) scores[(2 * t + 1) * a.tableBlocks + b] = k1;
                    } else if ((2 * t) % min(a.rowColumns, 8u) == 0u) {
                        const uint32_t i = 2 * t / min(a.rowColumns, 8u);
                        if (i >= i0 && i < i1) scores[i * a.tableBlocks + b] = k0;
                    }
                }
                if (__any_sync(0xFFFFFFFFu, lane < 16u && base + lane < end && page >= a.pageCount)) *a.errorFlag = kFlagPage;
            }
        }
    }
    __syncthreads();

    // ---- the lists, a row after the other ----
    for (uint32_t i = 0; i < rows; ++i) {
        const uint32_t seen = seenBlocks[i];
        uint32_t *out = a.ids + ((size_t)(row0 + i) * a.kvHeads + head) * a.blocks;
        if (seen <= a.blocks) {
            for (uint32_t k = tid; k < a.blocks; k += kSelectThreads) out[k] = k < seen ? k : FF_NO_SLOT;
            continue;
        }
        for (uint32_t k = tid; k < a.first; k += kSelectThreads) out[k] = k;
        for (uint32_t k = tid; k < a.last; k += kSelectThreads) out[a.blocks - a.last + k] = seen - a.last + k;
        if (!wanted) continue;
        const uint32_t *mine = scores + i * a.tableBlocks + a.first, n = seen - a.last - a.first;  // (more than wanted)
        // the largest bound that `wanted` scores reach: low is reached by that many, high is not
        uint32_t low = 0, high = 0, reached = n;
        uint32_t turn = 0;
        auto count = [&](uint32_t bound) {
            uint32_t c = 0;
            for (uint32_t k = tid; k < n; k += kSelectThreads) c += mine[k] >= bound;
            c = __reduce_add_sync(0xFFFFFFFFu, c);
            if (lane == 0) counts[turn][warp] = c;
            __syncthreads();
            c = __reduce_add_sync(0xFFFFFFFFu, lane < kSelectWarps ? counts[turn][lane] : 0u);
            turn ^= 1u;
            return c;
        };
        // (high = 0 stands for 2^32)
        while (reached != wanted && high - low != 1u) {
            const uint32_t mid = low + (uint32_t)(((high ? (unsigned long long)high : 1ull << 32) - low) >> 1);
            const uint32_t c = count(mid);
            if (c >= wanted) low = mid, reached = c;
            else high = mid;
        }
        // those above the bound, and the first of those at it
        const uint32_t each = (n + kSelectThreads - 1) / kSelectThreads * 32u, k0 = min(warp * each, n), k1 = min(k0 + each, n);
        uint32_t above = 0, at = 0;
        for (uint32_t k = k0; k < k1; k += 32) {
            const uint32_t v = k + lane < k1 ? mine[k + lane] : 0u;
            const bool there = k + lane < k1;
            above += __popc(__ballot_sync(0xFFFFFFFFu, there && v > low));
            at += __popc(__ballot_sync(0xFFFFFFFFu, there && v == low));
        }
        if (lane == 0) greater[warp] = above, equal[warp] = at;
        __syncthreads();
        uint32_t aboveBefore = 0, atBefore = 0, aboveAll = 0;
#pragma unroll
        for (uint32_t w = 0; w < kSelectWarps; ++w) {
            if (w < warp) aboveBefore += greater[w], atBefore += equal[w];
            aboveAll += greater[w];
        }
        const uint32_t ties = wanted - aboveAll;
        for (uint32_t k = k0; k < k1; k += 32) {
            const bool there = k + lane < k1;
            const uint32_t v = there ? mine[k + lane] : 0u;
            const uint32_t up = __ballot_sync(0xFFFFFFFFu, there && v > low), same = __ballot_sync(0xFFFFFFFFu, there && v == low), under = (1u << lane) - 1u;
            const uint32_t sameBefore = atBefore + __popc(same & under);
            if (there && (v > low || (v == low && sameBefore < ties))) out[a.first + aboveBefore + __popc(up & under) + min(sameBefore, ties)] = a.first + k + lane;
            aboveBefore += __popc(up);
            atBefore += __popc(same);
        }
        __syncthreads();  // (the counts are free for the next row)
    }
}

KernelSmemMemo selectMemo[3];

}  // namespace

bool launch_block_means(FFAttention *att, const uint8_t *pages, uint32_t pageCount, const uint32_t *blockTable, uint32_t tableStride, uint32_t tableKeys,
                        const uint32_t *oldLengths, const uint32_t *newLengths, uint32_t requests, uint16_t *means, cudaStream_t stream, const char **error) {
    const FFAttentionConfig &c = att->cfg;
    const MeansArgs args{pages, pageCount, blockTable, tableStride, tableKeys, oldLengths, newLengths, requests, c.kvHeads, (uint32_t)__builtin_ctz(c.pageTokens),
                         page_layout(c), means, att->errorFlag};
    const uint64_t most = ((uint64_t)requests * (tableKeys / kTileKeys) * c.kvHeads + kMeansThreads / 32 - 1) / (kMeansThreads / 32);
    const uint32_t grid = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(most, 4u * (uint32_t)att->smCount));
    auto launch = [&](auto kernel) { return launched(att, launch_pdl(kernel, dim3(grid), dim3(kMeansThreads), 0, stream, args), "k_block_means", error); };
    return c.headDim == 256 ? launch(k_block_means<256>) : c.headDim == 128 ? launch(k_block_means<128>) : launch(k_block_means<64>);
}

bool launch_select_blocks(FFAttention *att, const uint16_t *q, uint32_t qStride, uint32_t tokens, const uint16_t *means, uint32_t pageCount,
                          const uint32_t *blockTable, uint32_t tableStride, uint32_t tableBlocks, const uint32_t *rowStart, const uint32_t *lengths,
                          uint32_t requests, uint32_t blocks, uint32_t first, uint32_t last, uint32_t *ids, cudaStream_t stream, const char **error) {
    const FFAttentionConfig &c = att->cfg;
    const uint32_t group = c.heads / c.kvHeads;
    uint32_t rowColumns = group > 8 ? (group + 7u) & ~7u : 1u;
    while (rowColumns < group) rowColumns *= 2;
    // As many rows as a product has columns for, which then read the means once; one where the CTAs would not fill the GPU, and where
    // the scores would not leave room for two CTAs an SM.
    uint32_t rows = rowColumns < 8 ? kSelectRows / rowColumns : 1u;
    if ((uint64_t)tokens * c.kvHeads <= 2ull * att->smCount) rows = 1;
    while (rows > 1 && select_smem(c.headDim, 8, rows, tableBlocks) > 100u * 1024u) rows /= 2;
    const uint32_t columns = (rows * rowColumns + 7u) & ~7u, smem = select_smem(c.headDim, columns, rows, tableBlocks);
    const SelectArgs args{q, qStride, tokens, means, pageCount, blockTable, tableStride, tableBlocks, rowStart, lengths, requests, c.heads, c.kvHeads,
                          (uint32_t)__builtin_ctz(c.pageTokens), blocks, first, last, ids, rows, rowColumns, att->errorFlag};
    const dim3 grid((tokens + rows - 1) / rows, c.kvHeads);
    auto launch = [&](auto kernel, KernelSmemMemo &memo) {
        if (!memo.prepare(kernel, att->device, smem, kSelectThreads, nullptr, error)) return false;
        return launched(att, launch_pdl(kernel, grid, dim3(kSelectThreads), smem, stream, args), "k_select_blocks", error);
    };
    if (c.headDim == 256) return launch(k_select_blocks<256>, selectMemo[2]);
    if (c.headDim == 128) return launch(k_select_blocks<128>, selectMemo[1]);
    return launch(k_select_blocks<64>, selectMemo[0]);
}

}  // namespace ff

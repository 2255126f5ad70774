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

// Scores: the blocks' means times the rows' queries, 16 blocks a warp at a time on mma.sync.  Both factors are whole numbers of at
// most 7 bits times a power of two of their own (the means as they are held, the queries as they are staged), so that every sum is below 2^23 of
// its unit and exact in whatever order; the largest of a row's heads is the score.  Then the bound that as many scores reach as are
// wanted, two bits of it at a time, until the number that reaches it is the number wanted or all bits are known: of the scores at the
// bound the first are taken.
//
// Two forms.  k_select_split: a cluster of CTAs for each row and head, which share the blocks; the first of them gets the others' scores and
// makes the list.  k_select_rows: some neighbouring rows a CTA, which read the means of their request once; a warp makes a list.
constexpr int kSelectThreads = 256, kSelectWarps = kSelectThreads / 32;
constexpr uint32_t kSelectColumns = 64;  // of a CTA's product, at most
constexpr uint32_t kMostSplit = 8;       // CTAs of a cluster, at most

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
    uint32_t rows, rowColumns, columns;  // of a CTA; columns of a row: the heads of its group, to a power of two or a multiple of 8
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

// What a CTA knows of its rows.
struct SelectRows {
    uint32_t request[kSelectWarps], seen[kSelectWarps];  // of each row; blocks that it sees
    int exponents[kSelectColumns];                       // of a column's largest value; kNoNumber: it has a value that is not finite
    static constexpr int kNoNumber = -1000;
};
// the query of column c, or null: a row's columns are its heads, the last of them again in what is left
template <int DIM>
__device__ __forceinline__ const uint16_t *select_column(const SelectArgs &a, uint32_t row0, uint32_t rows, uint32_t head, uint32_t c) {
    const uint32_t i = c / a.rowColumns, group = a.heads / a.kvHeads;
    return i < rows ? a.q + (size_t)(row0 + i) * a.qStride + (size_t)(head * group + min(c % a.rowColumns, group - 1u)) * DIM : nullptr;
}
// Requests and blocks of the rows, and the columns' exponents; a barrier in front, which s.request and s.seen are cleared before, and one behind.
template <int DIM>
__device__ __forceinline__ void select_look_up(const SelectArgs &a, SelectRows &s, uint32_t row0, uint32_t rows, uint32_t head) {
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    for (uint32_t c = warp; c < a.columns; c += kSelectWarps) {
        const uint16_t *src = select_column<DIM>(a, row0, rows, head, c);
        uint32_t most = 0;
#pragma unroll
        for (uint32_t d = 2 * lane; d < DIM; d += 64)
            if (src) most = __vmaxu2(most, __ldg(reinterpret_cast<const uint32_t *>(src + d)) & 0x7FFF7FFFu);
        most = __reduce_max_sync(0xFFFFFFFFu, max(most & 0xFFFFu, most >> 16)) >> 7;
        if (lane == 0) s.exponents[c] = most == 255u ? SelectRows::kNoNumber : max((int)most - 127, -100);
    }
    for (uint32_t r = tid; r < a.requests; r += kSelectThreads) {
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
// The columns as they are multiplied: whole numbers of at most 7 bits at the exponents, times a power of two that a row's columns share.
template <int DIM>
__device__ __forceinline__ void select_stage(const SelectArgs &a, const SelectRows &s, uint32_t row0, uint32_t rows, uint32_t head, uint8_t *to) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    for (uint32_t c = warp; c < a.columns; c += kSelectWarps) {
        const uint16_t *src = select_column<DIM>(a, row0, rows, head, c);
        const uint32_t c0 = c / a.rowColumns * a.rowColumns;
        int top = -100;
        for (uint32_t k = lane; k < a.rowColumns; k += 32)
            if (c0 + k < a.columns) top = max(top, s.exponents[c0 + k]);
        top = __reduce_max_sync(0xFFFFFFFFu, top);
        const int mine = s.exponents[c], e = max(mine, top - 60);
        if (mine == SelectRows::kNoNumber) src = nullptr;  // (counts as zeros)
        const float down = power_of_two(6 - e), up = power_of_two(e - top);
#pragma unroll
        for (uint32_t d = 2 * lane; d < DIM; d += 64) {
            const uint32_t v = src ? __ldg(reinterpret_cast<const uint32_t *>(src + d)) : 0u;
            const float x = fminf(fmaxf(rintf(low16(v) * down), -127.0f), 127.0f) * up, y = fminf(fmaxf(rintf(high16(v) * down), -127.0f), 127.0f) * up;
            *reinterpret_cast<uint32_t *>(to + c * select_query_stride(DIM) + 2 * d) = pack_bf16x2(x, y);
        }
    }
}
// Scores of request r's blocks below `end`, in whole numbers of their order, to store(row of the CTA, block, score): sixteen at a time from
// 16 tile on, 16 step apart.
template <int DIM, typename Store>
__device__ __forceinline__ void select_score(const SelectArgs &a, const uint8_t *queries, uint32_t head, uint32_t r, uint32_t end, uint32_t tile, uint32_t step, Store store) {
    constexpr uint32_t kChunks = DIM / 32;
    const uint32_t lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u, perPage = max(1u, (1u << a.pageShift) >> kBlockShift);
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
        float best[4];  // [block g: column 2 t, 2 t + 1; block g + 8: likewise] of the columns so far that are the row's
        for (uint32_t n = 0; n < a.columns; n += 8) {
            float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (uint32_t c = 0; c < kChunks; ++c) {
                const uint4 b = *reinterpret_cast<const uint4 *>(queries + (n + g) * select_query_stride(DIM) + 64 * c + 16 * t);
                mma_bf16(acc, v[0][c].x, v[1][c].x, v[0][c].y, v[1][c].y, b.x, b.y);
                mma_bf16(acc, v[0][c].z, v[1][c].z, v[0][c].w, v[1][c].w, b.z, b.w);
            }
            const bool begins = a.rowColumns <= 8 || n % a.rowColumns == 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) best[k] = begins || acc[k] != acc[k] ? acc[k] : fmaxf(best[k], acc[k]);  // (a NaN mean makes all columns NaN)
            if (a.rowColumns > 8 && (n + 8) % a.rowColumns) continue;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t b = base + g + 8 * h, width = min(a.rowColumns, 8u);
                uint32_t k0 = order_of(best[2 * h]), k1 = order_of(best[2 * h + 1]);
                if (gone >> (g + 8 * h) & 1u) k0 = k1 = 0u;
                if (width > 1) k0 = max(k0, k1);
                if (width > 2) k0 = max(k0, __shfl_xor_sync(0xFFFFFFFFu, k0, 1));
                if (width > 4) k0 = max(k0, __shfl_xor_sync(0xFFFFFFFFu, k0, 2));
                if (b < end && (2 * t) % width == 0u) {
                    store((n + 2 * t) / a.rowColumns, b, k0);
                    if (width == 1) store(n + 2 * t + 1, b, k1);
                }
            }
        }
    }
}
// The bound: the largest number that at least `wanted` of n scores reach, or any that `wanted` of them do.  count(t, step): how many reach t + step,
// t + 2 step, t + 3 step.
template <typename Count>
__device__ __forceinline__ uint32_t select_bound(uint32_t n, uint32_t wanted, Count count) {
    uint32_t low = 0, reached = n;
    for (int shift = 30; shift >= 0 && reached != wanted; shift -= 2) {
        const uint3 c = count(low, 1u << shift);
        const uint32_t up = (c.x >= wanted) + (c.y >= wanted) + (c.z >= wanted);
        reached = up == 0 ? reached : up == 1 ? c.x : up == 2 ? c.y : c.z;
        low += up << shift;
    }
    return low;
}

template <int DIM>
__global__ void __launch_bounds__(kSelectThreads) k_select_split(const __grid_constant__ SelectArgs a) {
    extern __shared__ __align__(16) uint8_t selectSmem[];
    __shared__ SelectRows s;
    __shared__ uint4 counts[2][kSelectWarps];
    __shared__ uint32_t greater[kSelectWarps], equal[kSelectWarps];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const uint32_t head = blockIdx.z, row = blockIdx.y, cta = blockIdx.x, ctas = gridDim.x;
    uint32_t *scores = reinterpret_cast<uint32_t *>(selectSmem + a.columns * select_query_stride(DIM));  // those of the cluster's first CTA count
    if (tid == 0) s.request[0] = FF_NO_SLOT, s.seen[0] = 0u;
    pdl_enter();
    if (ctas > 1) cluster_sync_all();  // (the first CTA is there to be written to)
    else __syncthreads();
    select_look_up<DIM>(a, s, row, 1, head);
    __syncthreads();
    const uint32_t seen = s.seen[0], wanted = a.blocks - a.first - a.last;
    uint32_t *out = a.ids + ((size_t)row * a.kvHeads + head) * a.blocks;
    if (seen > a.blocks && wanted) {
        select_stage<DIM>(a, s, row, 1, head, selectSmem);
        __syncthreads();
        const uint32_t to = ctas > 1 ? map_to_cta(sm_addr(scores), 0) : 0u;
        select_score<DIM>(a, selectSmem, head, s.request[0], seen - a.last, cta * kSelectWarps + warp, ctas * kSelectWarps, [&](uint32_t i, uint32_t b, uint32_t score) {
            if (i) return;  // (a column of no row)
            if (ctas > 1) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to + 4 * b), "r"(score) : "memory");
            else scores[b] = score;
        });
    }
    if (ctas > 1) cluster_sync_all();
    else __syncthreads();
    if (cta) return;

    if (seen <= a.blocks) {
        for (uint32_t k = tid; k < a.blocks; k += kSelectThreads) out[k] = k < seen ? k : FF_NO_SLOT;
        return;
    }
    for (uint32_t k = tid; k < a.first; k += kSelectThreads) out[k] = k;
    for (uint32_t k = tid; k < a.last; k += kSelectThreads) out[a.blocks - a.last + k] = seen - a.last + k;
    if (!wanted) return;
    const uint32_t *mine = scores + a.first, n = seen - a.last - a.first;  // (more than wanted)
    uint32_t turn = 0;
    const uint32_t low = select_bound(n, wanted, [&](uint32_t t, uint32_t step) {
        uint3 c = make_uint3(0u, 0u, 0u);
#pragma unroll 4
        for (uint32_t k = tid; k < n; k += kSelectThreads) {
            const uint32_t v = mine[k];
            c.x += v >= t + step, c.y += v >= t + 2 * step, c.z += v >= t + 3 * step;
        }
        c.x = __reduce_add_sync(0xFFFFFFFFu, c.x), c.y = __reduce_add_sync(0xFFFFFFFFu, c.y), c.z = __reduce_add_sync(0xFFFFFFFFu, c.z);
        if (lane == 0) counts[turn][warp] = make_uint4(c.x, c.y, c.z, 0u);
        __syncthreads();
        c = make_uint3(0u, 0u, 0u);
#pragma unroll
        for (int w = 0; w < kSelectWarps; ++w) {
            const uint4 of = counts[turn][w];
            c.x += of.x, c.y += of.y, c.z += of.z;
        }
        turn ^= 1u;
        return c;
    });
    // those above the bound, and the first of those at it: a warp a run of the blocks
    const uint32_t each = (n + kSelectThreads - 1) / kSelectThreads * 32u, k0 = min(warp * each, n), k1 = min(k0 + each, n);
    uint32_t above = 0, at = 0;
    for (uint32_t k = k0 + lane; k < k1; k += 32) {
        above += mine[k] > low;
        at += mine[k] == low;
    }
    above = __reduce_add_sync(0xFFFFFFFFu, above), at = __reduce_add_sync(0xFFFFFFFFu, at);
    if (lane == 0) greater[warp] = above, equal[warp] = at;
    __syncthreads();
    uint32_t aboveBefore = 0, atBefore = 0, aboveAll = 0;
#pragma unroll
    for (uint32_t w = 0; w < kSelectWarps; ++w) {
        if (w < warp) aboveBefore += greater[w], atBefore += equal[w];
        aboveAll += greater[w];
    }
    const uint32_t ties = wanted - aboveAll, under = (1u << lane) - 1u;
    for (uint32_t k = k0; k < k1; k += 32) {
        const bool there = k + lane < k1;
        const uint32_t v = there ? mine[k + lane] : 0u;
        const uint32_t up = __ballot_sync(0xFFFFFFFFu, there && v > low), same = __ballot_sync(0xFFFFFFFFu, there && v == low);
        const uint32_t sameBefore = atBefore + __popc(same & under);
        if (there && (v > low || (v == low && sameBefore < ties))) out[a.first + aboveBefore + __popc(up & under) + min(sameBefore, ties)] = a.first + k + lane;
        aboveBefore += __popc(up);
        atBefore += __popc(same);
    }
}

template <int DIM>
__global__ void __launch_bounds__(kSelectThreads) k_select_rows(const __grid_constant__ SelectArgs a) {
    extern __shared__ __align__(16) uint8_t selectSmem[];
    __shared__ SelectRows s;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const uint32_t head = blockIdx.y, row0 = blockIdx.x * a.rows, rows = min(a.rows, a.tokens - row0);
    uint32_t *scores = reinterpret_cast<uint32_t *>(selectSmem + a.columns * select_query_stride(DIM));  // [rows][tableBlocks]
    if (tid < kSelectWarps) s.request[tid] = FF_NO_SLOT, s.seen[tid] = 0u;
    pdl_enter();
    __syncthreads();
    select_look_up<DIM>(a, s, row0, rows, head);
    __syncthreads();
    const uint32_t wanted = a.blocks - a.first - a.last;
    select_stage<DIM>(a, s, row0, rows, head, selectSmem);
    __syncthreads();
    for (uint32_t i0 = 0, i1; i0 < rows; i0 = i1) {  // request by request
        uint32_t end = 0;  // blocks that a row of the request may choose
        for (i1 = i0; i1 < rows && s.request[i1] == s.request[i0]; ++i1)
            if (s.seen[i1] > a.blocks) end = max(end, s.seen[i1] - a.last);
        if (s.request[i0] == FF_NO_SLOT || !wanted) continue;
        select_score<DIM>(a, selectSmem, head, s.request[i0], end, warp, kSelectWarps, [&](uint32_t i, uint32_t b, uint32_t score) {
            if (i >= i0 && i < i1) scores[i * a.tableBlocks + b] = score;
        });
    }
    __syncthreads();

    if (warp >= rows) return;
    const uint32_t seen = s.seen[warp];
    uint32_t *out = a.ids + ((size_t)(row0 + warp) * a.kvHeads + head) * a.blocks;
    if (seen <= a.blocks) {
        for (uint32_t k = lane; k < a.blocks; k += 32) out[k] = k < seen ? k : FF_NO_SLOT;
        return;
    }
    for (uint32_t k = lane; k < a.first; k += 32) out[k] = k;
    for (uint32_t k = lane; k < a.last; k += 32) out[a.blocks - a.last + k] = seen - a.last + k;
    if (!wanted) return;
    const uint32_t *mine = scores + warp * a.tableBlocks + a.first, n = seen - a.last - a.first;  // (more than wanted)
    const uint32_t low = select_bound(n, wanted, [&](uint32_t t, uint32_t step) {
        uint3 c = make_uint3(0u, 0u, 0u);
#pragma unroll 4
        for (uint32_t k = lane; k < n; k += 32) {
            const uint32_t v = mine[k];
            c.x += v >= t + step, c.y += v >= t + 2 * step, c.z += v >= t + 3 * step;
        }
        return make_uint3(__reduce_add_sync(0xFFFFFFFFu, c.x), __reduce_add_sync(0xFFFFFFFFu, c.y), __reduce_add_sync(0xFFFFFFFFu, c.z));
    });
    uint32_t above = 0;
    for (uint32_t k = lane; k < n; k += 32) above += mine[k] > low;
    const uint32_t ties = wanted - __reduce_add_sync(0xFFFFFFFFu, above), under = (1u << lane) - 1u;
    uint32_t aboveBefore = 0, atBefore = 0;
    for (uint32_t k = 0; k < n; k += 32) {
        const bool there = k + lane < n;
        const uint32_t v = there ? mine[k + lane] : 0u;
        const uint32_t up = __ballot_sync(0xFFFFFFFFu, there && v > low), same = __ballot_sync(0xFFFFFFFFu, there && v == low);
        const uint32_t sameBefore = atBefore + __popc(same & under);
        if (there && (v > low || (v == low && sameBefore < ties))) out[a.first + aboveBefore + __popc(up & under) + min(sameBefore, ties)] = a.first + k + lane;
        aboveBefore += __popc(up);
        atBefore += __popc(same);
    }
}

KernelSmemMemo selectMemo[2][3];

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
    const uint32_t group = c.heads / c.kvHeads, sms = (uint32_t)att->smCount;
    uint32_t rowColumns = group > 8 ? (group + 7u) & ~7u : 1u;
    while (rowColumns < group) rowColumns *= 2;
    SelectArgs args{q, qStride, tokens, means, pageCount, blockTable, tableStride, tableBlocks, rowStart, lengths, requests, c.heads, c.kvHeads,
                    (uint32_t)__builtin_ctz(c.pageTokens), blocks, first, last, ids, 1, rowColumns, 0, att->errorFlag};
    const uint64_t lists = (uint64_t)tokens * c.kvHeads;
    const int dim = c.headDim == 256 ? 2 : c.headDim == 128 ? 1 : 0;
    if (lists <= 4ull * sms) {
        // CTAs to fill the GPU, as long as each of them has eight warps' blocks
        uint32_t ctas = 1;
        while (ctas < kMostSplit && 2 * ctas * lists <= 2 * sms && 2 * ctas * kSelectWarps * 16 <= tableBlocks) ctas *= 2;
        args.columns = std::max(8u, rowColumns);
        const uint32_t smem = select_smem(c.headDim, args.columns, 1, tableBlocks);
        auto launch = [&](auto kernel) {
            if (!selectMemo[0][dim].prepare(kernel, att->device, smem, kSelectThreads, nullptr, error)) return false;
            cudaLaunchConfig_t config{};
            config.gridDim = dim3(ctas, tokens, c.kvHeads);
            config.blockDim = dim3(kSelectThreads);
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
        return dim == 2 ? launch(k_select_split<256>) : dim == 1 ? launch(k_select_split<128>) : launch(k_select_split<64>);
    }
    // A warp's list each, as far as the columns and the shared memory for their scores go.
    args.rows = std::min((uint32_t)kSelectWarps, kSelectColumns / rowColumns);
    while (args.rows > 1 && select_smem(c.headDim, std::max(8u, args.rows * rowColumns), args.rows, tableBlocks) > 100u * 1024u) args.rows /= 2;
    args.columns = (args.rows * rowColumns + 7u) & ~7u;
    const uint32_t smem = select_smem(c.headDim, args.columns, args.rows, tableBlocks);
    auto launch = [&](auto kernel) {
        if (!selectMemo[1][dim].prepare(kernel, att->device, smem, kSelectThreads, nullptr, error)) return false;
        return launched(att, launch_pdl(kernel, dim3((tokens + args.rows - 1) / args.rows, c.kvHeads), dim3(kSelectThreads), smem, stream, args), "k_select_rows", error);
    };
    return dim == 2 ? launch(k_select_rows<256>) : dim == 1 ? launch(k_select_rows<128>) : launch(k_select_rows<64>);
}

}  // namespace ff

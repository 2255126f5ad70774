// The paged INT4 key/value cache: its book-keeping from request lengths, rotary positions, quantizing append,
// read-back.
#include <algorithm>

#include "ff_attention.cuh"

namespace ff {

// ---- book-keeping ------------------------------------------------------------------------------

// One launch and no order between its CTAs: whatever a CTA needs of the others' work it works out itself.  Every CTA
// scans the requests (rows, pages taken, pages given back; a thread a run of them), then the CTAs share the rows, the
// pages and the table entries.  The k-th page taken is the k-th from the top of the stack as it stands with the
// returned pages on it; where that is a returned page its id is read from the table entry it came from, which
// nothing writes: a request either grows or shrinks.  So no value passes through memory that this launch writes.
// Entries that are no page (of requests for which none was left) do not go back.  A CTA that meets one among its share of those
// given back says so at the end, and the last CTA does all again with the pages alone counted.  (Looked for beforehand by every CTA
// they cost 1000 mixed requests 2.1 us, this way 0.8.)
// Bound by latency: two rounds of loads, a scan, a search of ten steps; 3.9 us for 16 requests of a decode step, 7.3 us for 1000
// requests that grow, shrink and end (in a graph; a call from Python is 8.5 us of the host's time).
constexpr int kPlanThreads = 1024;

struct PlanArgs {
    const uint32_t *oldLengths, *newLengths;
    uint32_t requests;
    uint32_t *blockTable;
    uint32_t tableStride;
    uint32_t *freePages;
    uint32_t pageCount;
    const uint32_t *freeCountIn;
    uint32_t *freeCountOut, *rowStart, *positions, *slots;
    uint32_t rows, pageShift;
    uint32_t *done, *errorFlag;
};

// Rows are counted up to here, what is more stays there: more than the arrays hold by far (2^24), and two counts add up in 32
// bits.  (A length that is none, as -1, would make the sums wrap.)  Pages are at most the table's entries, which are no more.
constexpr uint32_t kMost = 1u << 30;
__device__ __forceinline__ uint32_t add_counts(uint32_t a, uint32_t b) { return min(a + b, kMost); }

struct PlanRequest {
    uint32_t rows, had, has;  // new rows; pages before and after, as far as the table row goes
    uint32_t oldLength;
    bool cut;
    __device__ uint32_t taken() const { return has > had ? has - had : 0u; }
    __device__ uint32_t given() const { return had > has ? had - has : 0u; }
};
__device__ __forceinline__ PlanRequest plan_request(const PlanArgs &a, uint32_t r) {
    const uint32_t before = __ldg(a.oldLengths + r), after = __ldg(a.newLengths + r);
    const uint32_t mask = (1u << a.pageShift) - 1u;
    PlanRequest p;
    p.oldLength = before;
    p.rows = after > before ? min(after - before, kMost) : 0u;
    const uint32_t had = (before >> a.pageShift) + ((before & mask) != 0u), has = (after >> a.pageShift) + ((after & mask) != 0u);
    p.cut = had > a.tableStride || has > a.tableStride;
    p.had = min(had, a.tableStride);
    p.has = min(has, a.tableStride);
    return p;
}

// What every CTA knows: first row, page taken and page given back of every thread's run of requests, and behind the last.
struct PlanSums {
    uint32_t first[3][kPlanThreads + 1];
    uint32_t warpSum[3][32];
};
// The kind's sum over the CTA's threads before each of them; `own` the thread's.
__device__ __forceinline__ uint32_t warp_scan(uint32_t own, uint32_t *all) {
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t s = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, s, d);
        if (lane >= (uint32_t)d) s = add_counts(s, v);
    }
    if (lane == 31u) *all = s;
    const uint32_t front = __shfl_up_sync(0xFFFFFFFFu, s, 1);
    return lane ? front : 0u;
}
// the run that holds the n-th of a kind, n below its total
__device__ __forceinline__ uint32_t run_of(const uint32_t *first, uint32_t n) {
    uint32_t low = 0, high = kPlanThreads;  // first[low] <= n < first[high]
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint32_t mid = (low + high) >> 1;
        if (first[mid] <= n) low = mid;
        else high = mid;
    }
    return low;
}
// Rows, table entries and returned pages, shared among `step` threads.  kHoles: of the entries given back those alone count (in
// `first` too) that are pages.  Whether one that is none was met.
template <bool kHoles>
__device__ __forceinline__ bool plan_write(const PlanArgs &a, const PlanSums &s, uint32_t free, uint32_t run, uint32_t at, uint32_t step) {
    const uint32_t totalRows = s.first[0][kPlanThreads], totalTaken = s.first[1][kPlanThreads], totalGiven = s.first[2][kPlanThreads], height = free + totalGiven;
    // the page on place `place` of the stack with the returned pages on it
    auto stack_page = [&](uint32_t place) {
        if (place < free) return __ldg(a.freePages + place);
        uint32_t n = place - free;
        const uint32_t g = run_of(s.first[2], n);
        n -= s.first[2][g];
        for (uint32_t r = g * run;; ++r) {
            const PlanRequest p = plan_request(a, r);
            const uint32_t *entries = a.blockTable + (size_t)r * a.tableStride + p.has;
            if (!kHoles) {
                if (n < p.given()) return entries[n];
                n -= p.given();
            } else {
                for (uint32_t i = 0; i < p.given(); ++i)
                    if (entries[i] < a.pageCount && n-- == 0u) return entries[i];
            }
        }
    };
    auto taken_page = [&](uint32_t k) {
        const uint32_t place = height - 1u - k, page = k < height ? stack_page(place) : FF_NO_PAGE;
        if (page < a.pageCount) return page;
        if (k >= height || place < free) *a.errorFlag = kFlagNoPage;
        return FF_NO_PAGE;
    };
    for (uint32_t i = at; i < a.rows; i += step) {
        uint32_t position = 0, slot = FF_NO_SLOT;
        if (i < totalRows) {
            const uint32_t g = run_of(s.first[0], i);
            uint32_t n = i - s.first[0][g], taken = s.first[1][g];
            for (uint32_t r = g * run;; ++r) {
                const PlanRequest p = plan_request(a, r);
                if (n < p.rows) {
                    position = p.oldLength + n;
                    const uint32_t index = position >> a.pageShift;
                    uint32_t page = FF_NO_PAGE;
                    if (index < p.had) page = a.blockTable[(size_t)r * a.tableStride + index];
                    else if (index < p.has) page = taken_page(taken + index - p.had);
                    if (page < a.pageCount) slot = (page << a.pageShift) | (position & ((1u << a.pageShift) - 1u));
                    break;
                }
                n -= p.rows;
                taken += p.taken();
            }
        }
        a.positions[i] = position;
        a.slots[i] = slot;
    }
    for (uint32_t k = at; k < totalTaken; k += step) {
        const uint32_t g = run_of(s.first[1], k);
        uint32_t n = k - s.first[1][g];
        for (uint32_t r = g * run;; ++r) {
            const PlanRequest p = plan_request(a, r);
            if (n < p.taken()) {
                a.blockTable[(size_t)r * a.tableStride + p.had + n] = taken_page(k);
                break;
            }
            n -= p.taken();
        }
    }
    bool met = false;
    for (uint32_t k = at; k < totalGiven; k += step) {
        const uint32_t page = stack_page(free + k);
        met |= page >= a.pageCount;
        if (free + k < a.pageCount) a.freePages[free + k] = page;
    }
    return met;
}
// All of it by the last CTA, where entries that are no page were given back.
__device__ __noinline__ void plan_again(const PlanArgs &a, PlanSums &s, uint32_t free, uint32_t run) {
    const uint32_t t = threadIdx.x, warp = t >> 5;
    const uint32_t r0 = min(t * run, a.requests), r1 = min(r0 + run, a.requests);
    uint32_t own = 0;
    for (uint32_t r = r0; r < r1; ++r) {
        const PlanRequest p = plan_request(a, r);
        for (uint32_t i = 0; i < p.given(); ++i) own += a.blockTable[(size_t)r * a.tableStride + p.has + i] < a.pageCount;
    }
    const uint32_t front = warp_scan(own, &s.warpSum[2][warp]);
    __syncthreads();
    uint32_t before = 0, total = 0;
    for (uint32_t w = 0; w < 32u; ++w) {
        if (w == warp) before = total;
        total += s.warpSum[2][w];
    }
    s.first[2][t] = before + front;
    if (t == 0) s.first[2][kPlanThreads] = total;
    __syncthreads();
    plan_write<true>(a, s, free, run, t, kPlanThreads);
}

__global__ void __launch_bounds__(kPlanThreads) k_cache_plan(const __grid_constant__ PlanArgs a) {
    __shared__ PlanSums s;
    __shared__ uint32_t last, again;
    const uint32_t t = threadIdx.x, lane = t & 31u, warp = t >> 5;
    const uint32_t run = (a.requests + kPlanThreads - 1) / kPlanThreads;
    const uint32_t r0 = min(t * run, a.requests), r1 = min(r0 + run, a.requests);
    pdl_enter();
    const uint32_t free = min(__ldg(a.freeCountIn), a.pageCount);

    uint32_t sum[3] = {0u, 0u, 0u};
    bool cut = false;
    for (uint32_t r = r0; r < r1; ++r) {
        const PlanRequest p = plan_request(a, r);
        sum[0] = add_counts(sum[0], p.rows);
        sum[1] += p.taken();
        sum[2] += p.given();
        cut |= p.cut;
    }
    uint32_t before[3];  // sums over the warp's lanes before this one
#pragma unroll
    for (int i = 0; i < 3; ++i) before[i] = warp_scan(sum[i], &s.warpSum[i][warp]);
    __syncthreads();
    if (warp < 3u) s.warpSum[warp][lane] = warp_scan(s.warpSum[warp][lane], &s.first[warp][kPlanThreads]);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) s.first[i][t] = add_counts(s.warpSum[i][warp], before[i]);
    __syncthreads();

    const bool met = plan_write<false>(a, s, free, run, blockIdx.x * kPlanThreads + t, gridDim.x * kPlanThreads);
    if (blockIdx.x == 0) {
        uint32_t row = s.first[0][t];
        for (uint32_t r = r0; r < r1; ++r) {
            a.rowStart[r] = row;
            row = add_counts(row, plan_request(a, r).rows);
        }
        if (t == 0) a.rowStart[a.requests] = s.first[0][kPlanThreads];
        if (cut) *a.errorFlag = kFlagTableRow;
        if (t == 0 && s.first[0][kPlanThreads] > a.rows) *a.errorFlag = kFlagRows;
    }
    // the stack's height may go back to the word it came from: written when every CTA has read that
    const bool some = __syncthreads_or(met);
    if (t == 0) {
        if (s.first[2][kPlanThreads]) __threadfence();  // (what this CTA wrote comes before what the last one may write over it)
        const uint32_t n = atomicAdd(a.done, some ? 0x10001u : 1u);
        last = (n & 0xFFFFu) == gridDim.x - 1u;
        again = some || n >> 16;
        if (again) __threadfence();
    }
    __syncthreads();
    if (!last) return;
    if (again) plan_again(a, s, free, run);
    if (t == 0) {
        const uint32_t height = free + s.first[2][kPlanThreads], taken = s.first[1][kPlanThreads];
        *a.done = 0u;
        *a.freeCountOut = height > taken ? min(height - taken, a.pageCount) : 0u;
    }
}

static uint32_t shift_of(uint32_t pageTokens) { return (uint32_t)__builtin_ctz(pageTokens); }

bool launch_cache_plan(FFAttention *att, const uint32_t *oldLengths, const uint32_t *newLengths, uint32_t requests, uint32_t *blockTable,
                       uint32_t tableStride, uint32_t *freePages, uint32_t pageCount, const uint32_t *freeCountIn, uint32_t *freeCountOut,
                       uint32_t *rowStart, uint32_t *positions, uint32_t *slots, uint32_t rows, cudaStream_t stream, const char **error) {
    PlanArgs a{oldLengths, newLengths, requests, blockTable, tableStride, freePages, pageCount, freeCountIn, freeCountOut,
               rowStart, positions, slots, rows, shift_of(att->cfg.pageTokens), att->planCount, att->errorFlag};
    const uint32_t grid = std::max(1u, std::min((rows + kPlanThreads - 1) / kPlanThreads, (uint32_t)att->smCount));
    return launched(att, launch_pdl(k_cache_plan, dim3(grid), dim3(kPlanThreads), 0, stream, a), "k_cache_plan", error);
}

// ---- rotary positions --------------------------------------------------------------------------

__global__ void k_rope_table(const FFRopeConfig c, float2 *table, uint32_t positions) {
    const uint32_t half = c.rotaryDim / 2;
    const size_t total = (size_t)positions * half;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (size_t)gridDim.x * blockDim.x) {
        const uint32_t position = (uint32_t)(i / half), pair = (uint32_t)(i % half);
        double frequency = pow(c.base, -2.0 * pair / c.rotaryDim);
        if (c.scaling == FF_ROPE_LINEAR) frequency /= c.factor;
        if (c.scaling == FF_ROPE_BY_PARTS) {
            const double turns = c.originalContext * frequency / (2.0 * 3.14159265358979323846);
            const double kept = fmin(1.0, fmax(0.0, (turns - c.lowTurns) / (c.highTurns - c.lowTurns)));
            frequency *= kept + (1.0 - kept) / c.factor;
        }
        const double amplitude = c.amplitude == 0.0 ? 1.0 : c.amplitude;
        double s, co;
        sincos(position * frequency, &s, &co);
        table[i] = make_float2((float)(co * amplitude), (float)(s * amplitude));
    }
}

bool launch_rope_table(FFAttention *att, const FFRopeConfig &config, float *table, uint32_t positions, cudaStream_t stream, const char **error) {
    if (positions == 0 || config.rotaryDim == 0) return true;
    const size_t total = (size_t)positions * (config.rotaryDim / 2);
    const uint32_t grid = (uint32_t)std::min<size_t>((total + 255) / 256, (size_t)att->smCount * 16);
    k_rope_table<<<grid, 256, 0, stream>>>(config, reinterpret_cast<float2 *>(table), positions);
    return launched(att, cudaSuccess, "k_rope_table", error);
}

struct RopeArgs {
    RopeRows rows;
    const float *table;
    uint32_t tablePositions, rotaryDim;
    const uint32_t *positions, *slots;
    uint32_t tokens, unitsPerToken, headsPerUnit, kvHeads;
    uint8_t *pages;
    uint32_t slotCount, pageShift;
    PageLayout page;
    uint32_t *errorFlag;
};

__device__ __forceinline__ float bf16_low(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float bf16_high(uint32_t pair) { return __uint_as_float(pair & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// the lesser, the greater of two pairs of bf16; NaN if either is
__device__ __forceinline__ uint32_t min_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// A warp takes 256 values at a time, 256 / DIM heads of one row, eight values a lane, BATCH such steps' loads in flight.  Its
// cosines and sines stay in registers for all the heads it takes.  Bound by issue slots and the bytes of the rows together: 4096 rows
// of 16 query and 2 x 8 key/value heads of 256 are 113 MB and take 29.6 us (3.8 TB/s, 58 % of a copy's rate) at 62 % of the issue
// slots, 175 warp instructions for 256 values.  Two steps' loads in flight at 64 registers 29.6 us; four at 64 registers 38.3, four at 92
// (a quarter of the SM's warps) 38.9.
template <int DIM, bool INTERLEAVED, int BATCH>
__global__ void __launch_bounds__(128, 8) k_rope_rows(const RopeArgs a) {
    constexpr uint32_t kLanes = DIM / 8, kHeads = 32 / kLanes;
    const uint32_t lane = threadIdx.x & 31u, inHead = lane % kLanes, headInWarp = lane / kLanes;
    const uint32_t unit = blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5);
    const uint32_t token = unit / a.unitsPerToken, part = unit - token * a.unitsPerToken;
    pdl_enter();
    if (token >= a.tokens) return;
    const uint32_t qHeads = a.rows.q ? a.rows.qHeads : 0u, kEnd = qHeads + (a.rows.k ? a.kvHeads : 0u), allHeads = 2u * kEnd - qHeads;
    const uint32_t firstHead = part * a.headsPerUnit, endHead = min(firstHead + a.headsPerUnit, allHeads);

    // where head h of the row lies: queries, keys, values
    auto source = [&](uint32_t h) {
        const uint16_t *src = h < qHeads ? a.rows.q + (size_t)token * a.rows.qStride + h * DIM
                              : h < kEnd ? a.rows.k + (size_t)token * a.rows.kStride + (h - qHeads) * DIM
                                         : a.rows.v + (size_t)token * a.rows.vStride + (h - kEnd) * DIM;
        return *reinterpret_cast<const uint4 *>(src + inHead * 8u);  // (qOut may be q: no read-only load)
    };
    uint4 loaded[BATCH];
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
        const uint32_t h = firstHead + b * kHeads + headInWarp;
        loaded[b] = h < endHead ? source(h) : make_uint4(0u, 0u, 0u, 0u);
    }
    const uint32_t slot = a.slots ? __ldg(a.slots + token) : 0u;
    float c[8], s[8];
    const uint32_t half = a.rotaryDim / 2;
    const bool turns = inHead * 8u < a.rotaryDim, second = !INTERLEAVED && inHead * 8u >= half;
    if (turns) {
        uint32_t position = __ldg(a.positions + token);
        if (position >= a.tablePositions) {
            if (lane == 0) *a.errorFlag = kFlagPosition;
            position = 0;
        }
        const float4 *row = reinterpret_cast<const float4 *>(a.table + (size_t)position * a.rotaryDim) + (INTERLEAVED ? inHead * 2 : (inHead * 8u - (second ? half : 0u)) / 2);
#pragma unroll
        for (int i = 0; i < (INTERLEAVED ? 2 : 4); ++i) {
            const float4 v = __ldg(row + i);
            c[2 * i] = v.x, s[2 * i] = v.y, c[2 * i + 1] = v.z, s[2 * i + 1] = v.w;
        }
        if (!INTERLEAVED && !second)
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] = -s[i];  // a c - b s for the first of a pair, b c + a s for the second
    }
    const uint32_t inPage = slot & (a.page.pageTokens - 1u);
    uint8_t *page = a.pages + (uint64_t)(slot >> a.pageShift) * a.page.pageBytes;
    const bool placed = slot < a.slotCount;
    if (!placed && slot != FF_NO_SLOT && endHead > qHeads && lane == 0) *a.errorFlag = kFlagPage;

    for (uint32_t h0 = firstHead; h0 < endHead; h0 += BATCH * kHeads) {
        uint4 now[BATCH];
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            now[b] = loaded[b];
            const uint32_t h = h0 + (BATCH + b) * kHeads + headInWarp;
            if (h < endHead) loaded[b] = source(h);
        }
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const uint32_t h = h0 + b * kHeads + headInWarp;
            if (h0 + b * kHeads >= endHead) break;
            const bool live = h < endHead, isQ = h < qHeads, isK = !isQ && h < kEnd;
            uint32_t x[4] = {now[b].x, now[b].y, now[b].z, now[b].w};
            const bool rotates = turns && (isQ || isK);
            if (INTERLEAVED) {
                if (rotates) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p = bf16_low(x[i]), q = bf16_high(x[i]);
                        x[i] = pack_bf16(__fsub_rn(__fmul_rn(p, c[i]), __fmul_rn(q, s[i])), __fadd_rn(__fmul_rn(p, s[i]), __fmul_rn(q, c[i])));
                    }
                }
            } else if (__any_sync(0xFFFFFFFFu, rotates)) {
                // the partner's values lie rotaryDim / 16 lanes away
                const uint32_t away = half / 8u, from = turns ? (second ? lane - away : lane + away) : lane;
                uint32_t y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = __shfl_sync(0xFFFFFFFFu, x[i], from);
                if (rotates) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float o[2];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float own = j ? bf16_high(x[i]) : bf16_low(x[i]), other = j ? bf16_high(y[i]) : bf16_low(y[i]);
                            o[j] = __fadd_rn(__fmul_rn(own, c[2 * i + j]), __fmul_rn(other, s[2 * i + j]));
                        }
                        x[i] = pack_bf16(o[0], o[1]);
                    }
                }
            }
            if (live && isQ)
                *reinterpret_cast<uint4 *>(a.rows.qOut + (size_t)token * a.rows.qOutStride + h * DIM + inHead * 8u) = make_uint4(x[0], x[1], x[2], x[3]);
            // keys and values: quantized, eight lanes a group
            if (__any_sync(0xFFFFFFFFu, live && !isQ)) {
                uint32_t least = min_bf16x2(min_bf16x2(x[0], x[1]), min_bf16x2(x[2], x[3])), most = max_bf16x2(max_bf16x2(x[0], x[1]), max_bf16x2(x[2], x[3]));
#pragma unroll
                for (int d = 1; d < 8; d <<= 1) {
                    least = min_bf16x2(least, __shfl_xor_sync(0xFFFFFFFFu, least, d));
                    most = max_bf16x2(most, __shfl_xor_sync(0xFFFFFFFFu, most, d));
                }
                const uint32_t both = min_bf16x2(least, least >> 16), top = max_bf16x2(most, most >> 16);  // (their low halves)
                const float low = bf16_low(both), high = bf16_low(top);
                const uint32_t scaleBits = pack_bf16(__fdiv_rn(__fsub_rn(high, low), 15.0f), low);  // scale | bias
                const float scale = bf16_low(scaleBits);
                // a value that is no number is the minimum or the maximum, or makes both NaN, and the range with them
                const bool finite = scale < INFINITY;
                const float inverse = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
                float code[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) code[i] = __fmul_rn(__fsub_rn(i % 2 ? bf16_high(x[i / 2]) : bf16_low(x[i / 2]), low), inverse);
                // The scale is within 2^-9 of a fifteenth of the range, so no code reaches 15.5, but for scales without all their
                // bits or with a reciprocal that overflows (0 * inf stays below code 0, the rest is code 15).
                if (__any_sync(0xFFFFFFFFu, scale < 0x1p-118f))
#pragma unroll
                    for (int i = 0; i < 8; ++i) code[i] = fminf(fmaxf(code[i], 0.0f), 15.0f);
                // rounded to whole numbers by adding 1.5 * 2^23, whose bits add up to a constant
                uint32_t word = 0u;
#pragma unroll
                for (int i = 7; i >= 0; --i) word = word * 16u + __float_as_uint(__fadd_rn(code[i], 12582912.0f));
                word -= 0x4B400000u * 0x11111111u;
                if (live && !isQ && placed) {
                    uint8_t *block = page + (uint64_t)(isK ? h - qHeads : h - kEnd) * a.page.blockBytes + (isK ? 0u : a.page.values);
                    *reinterpret_cast<uint32_t *>(block + inPage * a.page.codeBytes + inHead * 4u) = finite ? word : 0u;
                    if ((inHead & 7u) == 0u)
                        *reinterpret_cast<uint32_t *>(block + a.page.keyWords + inPage * a.page.wordBytes + (inHead >> 3) * 4u) = finite ? scaleBits : 0x7FC07FC0u;
                }
            }
        }
    }
}

template <int DIM>
static cudaError_t start_rope(const RopeArgs &a, bool interleaved, bool many, dim3 grid, cudaStream_t stream) {
    const dim3 block(128);
    if (many) return interleaved ? launch_pdl(k_rope_rows<DIM, true, 2>, grid, block, 0, stream, a) : launch_pdl(k_rope_rows<DIM, false, 2>, grid, block, 0, stream, a);
    return interleaved ? launch_pdl(k_rope_rows<DIM, true, 1>, grid, block, 0, stream, a) : launch_pdl(k_rope_rows<DIM, false, 1>, grid, block, 0, stream, a);
}

bool launch_rope_rows(FFAttention *att, const RopeRows &rows, const FFRope &rope, const uint32_t *positions, const uint32_t *slots,
                      uint32_t tokens, uint8_t *pages, uint32_t pageCount, cudaStream_t stream, const char **error) {
    if (tokens == 0) return true;
    const FFAttentionConfig &cfg = att->cfg;
    RopeArgs a{};
    a.rows = rows;
    a.table = rope.table;
    a.tablePositions = rope.positions;
    a.rotaryDim = rope.rotaryDim;
    a.positions = positions;
    a.slots = slots;
    a.tokens = tokens;
    a.kvHeads = cfg.kvHeads;
    a.pages = pages;
    a.slotCount = pageCount * cfg.pageTokens;
    a.pageShift = shift_of(cfg.pageTokens);
    a.page = page_layout(cfg);
    a.errorFlag = att->errorFlag;
    const uint32_t perWarp = 256u / cfg.headDim;
    const uint32_t heads = (rows.q ? rows.qHeads : 0u) + (rows.k ? 2u * cfg.kvHeads : 0u);
    // Steps of a warp: as many as leave every SM 32 warps, up to eight.
    uint32_t steps = 1;
    while (steps < 8 && (uint64_t)tokens * ((heads + 2 * steps * perWarp - 1) / (2 * steps * perWarp)) >= (uint64_t)att->smCount * 32) steps *= 2;
    a.headsPerUnit = steps * perWarp;
    a.unitsPerToken = (heads + a.headsPerUnit - 1) / a.headsPerUnit;
    const dim3 grid((uint32_t)(((uint64_t)tokens * a.unitsPerToken + 3) / 4));
    const bool interleaved = rope.layout == FF_ROPE_INTERLEAVED;
    const cudaError_t st = cfg.headDim == 64 ? start_rope<64>(a, interleaved, steps > 1, grid, stream)
                           : cfg.headDim == 128 ? start_rope<128>(a, interleaved, steps > 1, grid, stream) : start_rope<256>(a, interleaved, steps > 1, grid, stream);
    return launched(att, st, "k_rope_rows", error);
}

// ---- read-back ---------------------------------------------------------------------------------

struct ReadArgs {
    const uint8_t *pages;
    const uint32_t *slots;
    uint16_t *k, *v;
    uint32_t tokens, kvHeads, slotCount, pageShift, unitsPerToken;
    PageLayout page;
    uint32_t *errorFlag;
};

// A warp takes 256 values at a time of one row, eight a lane, four such steps.  Bound by the bytes written: 4096 rows of 2 x 8 heads of
// 256, 43 MB, in 8.6 us (5.0 TB/s).
template <int DIM>
__global__ void __launch_bounds__(128) k_cache_read(const ReadArgs a) {
    constexpr uint32_t kLanes = DIM / 8, kHeads = 32 / kLanes, kSteps = 4;
    const uint32_t lane = threadIdx.x & 31u, inHead = lane % kLanes, headInWarp = lane / kLanes;
    const uint32_t unit = blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5);
    const uint32_t token = unit / a.unitsPerToken, part = unit - token * a.unitsPerToken;
    pdl_enter();
    if (token >= a.tokens) return;
    const uint32_t keys = a.k ? a.kvHeads : 0u, all = keys + (a.v ? a.kvHeads : 0u);
    const uint32_t slot = __ldg(a.slots + token), inPage = slot & (a.page.pageTokens - 1u);
    const uint8_t *page = a.pages + (uint64_t)(slot >> a.pageShift) * a.page.pageBytes;
    const bool placed = slot < a.slotCount;
    if (!placed && slot != FF_NO_SLOT && lane == 0) *a.errorFlag = kFlagPage;
    uint32_t w[kSteps], sb[kSteps];
#pragma unroll
    for (uint32_t i = 0; i < kSteps; ++i) {
        const uint32_t h = (part * kSteps + i) * kHeads + headInWarp;
        w[i] = sb[i] = 0u;
        if (h < all && placed) {
            const uint8_t *block = page + (uint64_t)(h < keys ? h : h - keys) * a.page.blockBytes + (h < keys ? 0u : a.page.values);
            w[i] = *reinterpret_cast<const uint32_t *>(block + inPage * a.page.codeBytes + inHead * 4u);
            sb[i] = *reinterpret_cast<const uint32_t *>(block + a.page.keyWords + inPage * a.page.wordBytes + (inHead >> 3) * 4u);
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < kSteps; ++i) {
        const uint32_t h = (part * kSteps + i) * kHeads + headInWarp;
        if (h >= all) break;
        const float scale = bf16_low(sb[i]), bias = bf16_high(sb[i]);
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = __fadd_rn(__fmul_rn((float)((w[i] >> (4 * j)) & 15u), scale), bias);
        uint16_t *out = (h < keys ? a.k : a.v) + ((uint64_t)token * a.kvHeads + (h < keys ? h : h - keys)) * DIM;
        *reinterpret_cast<uint4 *>(out + inHead * 8u) = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
    }
}

bool launch_cache_read(FFAttention *att, const uint8_t *pages, uint32_t pageCount, const uint32_t *slots, uint32_t tokens, uint16_t *k,
                       uint16_t *v, cudaStream_t stream, const char **error) {
    if (tokens == 0 || (!k && !v)) return true;
    const FFAttentionConfig &cfg = att->cfg;
    const uint32_t perUnit = 4u * 256u / cfg.headDim, heads = cfg.kvHeads * ((k ? 1u : 0u) + (v ? 1u : 0u));
    ReadArgs a{pages, slots, k, v, tokens, cfg.kvHeads, pageCount * cfg.pageTokens, shift_of(cfg.pageTokens), (heads + perUnit - 1) / perUnit, page_layout(cfg), att->errorFlag};
    const dim3 grid((uint32_t)(((uint64_t)tokens * a.unitsPerToken + 3) / 4)), block(128);
    const cudaError_t st = cfg.headDim == 64 ? launch_pdl(k_cache_read<64>, grid, block, 0, stream, a)
                           : cfg.headDim == 128 ? launch_pdl(k_cache_read<128>, grid, block, 0, stream, a) : launch_pdl(k_cache_read<256>, grid, block, 0, stream, a);
    return launched(att, st, "k_cache_read", error);
}

}  // namespace ff

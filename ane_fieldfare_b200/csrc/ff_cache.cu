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
// Bound by latency: two rounds of loads, a scan, a search of eleven steps.
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
    p.rows = after > before ? after - before : 0u;
    const uint32_t had = (before >> a.pageShift) + ((before & mask) != 0u), has = (after >> a.pageShift) + ((after & mask) != 0u);
    p.cut = had > a.tableStride || has > a.tableStride;
    p.had = min(had, a.tableStride);
    p.has = min(has, a.tableStride);
    return p;
}

__global__ void __launch_bounds__(kPlanThreads) k_cache_plan(const PlanArgs a) {
    // first row, page taken and page given back of every thread's run of requests, and behind the last
    __shared__ uint32_t first[3][kPlanThreads + 1];
    __shared__ uint32_t warpSum[3][32];
    __shared__ bool last;
    const uint32_t t = threadIdx.x, lane = t & 31u, warp = t >> 5;
    const uint32_t run = (a.requests + kPlanThreads - 1) / kPlanThreads;
    const uint32_t r0 = min(t * run, a.requests), r1 = min(r0 + run, a.requests);
    pdl_enter();
    const uint32_t free = min(__ldg(a.freeCountIn), a.pageCount);

    uint32_t sum[3] = {0u, 0u, 0u};
    bool cut = false;
    for (uint32_t r = r0; r < r1; ++r) {
        const PlanRequest p = plan_request(a, r);
        sum[0] += p.rows;
        sum[1] += p.taken();
        sum[2] += p.given();
        cut |= p.cut;
    }
    uint32_t scan[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        scan[i] = sum[i];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, scan[i], d);
            if (lane >= (uint32_t)d) scan[i] += v;
        }
        if (lane == 31u) warpSum[i][warp] = scan[i];
    }
    __syncthreads();
    if (warp < 3u) {
        uint32_t v = warpSum[warp][lane], s = v;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t u = __shfl_up_sync(0xFFFFFFFFu, s, d);
            if (lane >= (uint32_t)d) s += u;
        }
        warpSum[warp][lane] = s - v;
        if (lane == 31u) first[warp][kPlanThreads] = s;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) first[i][t] = warpSum[i][warp] + scan[i] - sum[i];
    __syncthreads();
    const uint32_t totalRows = first[0][kPlanThreads], totalTaken = first[1][kPlanThreads], totalGiven = first[2][kPlanThreads];

    // the run that holds the n-th of a kind, n below its total
    auto run_of = [&](int kind, uint32_t n) {
        uint32_t low = 0, high = kPlanThreads;  // first[low] <= n < first[high]
#pragma unroll
        for (int i = 0; i < 10; ++i) {
            const uint32_t mid = (low + high) >> 1;
            if (first[kind][mid] <= n) low = mid;
            else high = mid;
        }
        return low;
    };
    // the page on place `at` of the stack with the returned pages on it
    auto stack_page = [&](uint32_t at) {
        if (at < free) return __ldg(a.freePages + at);
        uint32_t n = at - free;
        const uint32_t g = run_of(2, n);
        n -= first[2][g];
        for (uint32_t r = g * run;; ++r) {
            const PlanRequest p = plan_request(a, r);
            if (n < p.given()) return a.blockTable[(size_t)r * a.tableStride + p.has + n];
            n -= p.given();
        }
    };
    const uint32_t height = free + totalGiven;
    auto taken_page = [&](uint32_t k) { return k < height ? stack_page(height - 1u - k) : FF_NO_PAGE; };

    const uint32_t at = blockIdx.x * kPlanThreads + t, step = gridDim.x * kPlanThreads;
    for (uint32_t i = at; i < a.rows; i += step) {
        uint32_t position = 0, slot = FF_NO_SLOT;
        if (i < totalRows) {
            const uint32_t g = run_of(0, i);
            uint32_t n = i - first[0][g], taken = first[1][g];
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
        const uint32_t g = run_of(1, k);
        uint32_t n = k - first[1][g];
        for (uint32_t r = g * run;; ++r) {
            const PlanRequest p = plan_request(a, r);
            if (n < p.taken()) {
                a.blockTable[(size_t)r * a.tableStride + p.had + n] = taken_page(k);
                break;
            }
            n -= p.taken();
        }
    }
    for (uint32_t k = at; k < totalGiven; k += step)
        if (free + k < a.pageCount) a.freePages[free + k] = stack_page(free + k);
    if (blockIdx.x == 0) {
        uint32_t row = first[0][t];
        for (uint32_t r = r0; r < r1; ++r) {
            a.rowStart[r] = row;
            row += plan_request(a, r).rows;
        }
        if (t == 0) a.rowStart[a.requests] = totalRows;
        if (cut) *a.errorFlag = kFlagTableRow;
        if (t == 0 && totalTaken > height) *a.errorFlag = kFlagNoPage;
        if (t == 0 && totalRows > a.rows) *a.errorFlag = kFlagRows;
    }
    // the stack's height may go back to the word it came from: written when every CTA has read that
    __syncthreads();
    if (t == 0) last = atomicAdd(a.done, 1u) == gridDim.x - 1u;
    __syncthreads();
    if (last && t == 0) {
        *a.done = 0u;
        *a.freeCountOut = height > totalTaken ? min(height - totalTaken, a.pageCount) : 0u;
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

// A warp takes 256 values at a time: 256 / DIM heads of one row, eight values a lane.  Its cosines and sines stay in
// registers for all the heads it takes.  Bound by the bytes of the rows.
template <int DIM, bool INTERLEAVED>
__global__ void __launch_bounds__(128) k_rope_rows(const RopeArgs a) {
    constexpr uint32_t kLanes = DIM / 8, kHeads = 32 / kLanes;
    const uint32_t lane = threadIdx.x & 31u, inHead = lane % kLanes, headInWarp = lane / kLanes;
    const uint32_t unit = blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5);
    const uint32_t token = unit / a.unitsPerToken, part = unit % a.unitsPerToken;
    pdl_enter();
    if (token >= a.tokens) return;
    const uint32_t qHeads = a.rows.q ? a.rows.qHeads : 0u, kHeadsTotal = a.rows.k ? a.kvHeads : 0u;
    const uint32_t allHeads = qHeads + 2u * kHeadsTotal;
    const uint32_t slot = a.slots ? __ldg(a.slots + token) : 0u;

    float c[8], s[8];
    const bool turns = inHead * 8u < a.rotaryDim;
    if (turns) {
        uint32_t position = __ldg(a.positions + token);
        if (position >= a.tablePositions) {
            if (lane == 0) *a.errorFlag = kFlagPosition;
            position = 0;
        }
        const uint32_t half = a.rotaryDim / 2;
        const float4 *row = reinterpret_cast<const float4 *>(a.table + (size_t)position * a.rotaryDim);
        if (INTERLEAVED) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float4 v = __ldg(row + inHead * 2 + i);
                c[2 * i] = v.x, s[2 * i] = v.y, c[2 * i + 1] = v.z, s[2 * i + 1] = v.w;
            }
        } else {
            const uint32_t first = inHead * 8u % half;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 v = __ldg(row + first / 2 + i);
                c[2 * i] = v.x, s[2 * i] = v.y, c[2 * i + 1] = v.z, s[2 * i + 1] = v.w;
            }
        }
    }
    const uint32_t firstHead = part * a.headsPerUnit, endHead = min(firstHead + a.headsPerUnit, allHeads);
    for (uint32_t h0 = firstHead; h0 < endHead; h0 += kHeads) {
        const uint32_t h = h0 + headInWarp;
        const bool live = h < endHead;
        const bool isQ = h < qHeads, isK = !isQ && h < qHeads + kHeadsTotal;
        const uint32_t head = isQ ? h : isK ? h - qHeads : h - qHeads - kHeadsTotal;
        uint32_t x[4] = {0u, 0u, 0u, 0u};
        if (live) {
            const uint16_t *src = isQ ? a.rows.q + (size_t)token * a.rows.qStride
                                      : isK ? a.rows.k + (size_t)token * a.rows.kStride : a.rows.v + (size_t)token * a.rows.vStride;
            const uint4 v = *reinterpret_cast<const uint4 *>(src + head * DIM + inHead * 8u);  // (qOut may be q)
            x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
        }
        const bool rotates = turns && (isQ || isK);
        if (INTERLEAVED) {
            if (rotates) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = bf16_low(x[i]), q = bf16_high(x[i]);
                    x[i] = pack_bf16(__fsub_rn(__fmul_rn(p, c[i]), __fmul_rn(q, s[i])), __fadd_rn(__fmul_rn(p, s[i]), __fmul_rn(q, c[i])));
                }
            }
        } else {
            // the partner's values lie rotaryDim / 16 lanes away
            const uint32_t half = a.rotaryDim / 2, away = half / 8u;
            const bool second = inHead * 8u >= half;
            const uint32_t from = turns ? (second ? lane - away : lane + away) : lane;
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
                        const float cs = __fmul_rn(own, c[2 * i + j]), sn = __fmul_rn(other, s[2 * i + j]);
                        o[j] = second ? __fadd_rn(sn, cs) : __fsub_rn(cs, sn);
                    }
                    x[i] = pack_bf16(o[0], o[1]);
                }
            }
        }
        if (live && isQ)
            *reinterpret_cast<uint4 *>(a.rows.qOut + (size_t)token * a.rows.qOutStride + head * DIM + inHead * 8u) = make_uint4(x[0], x[1], x[2], x[3]);
        // keys and values: quantized, eight lanes a group
        if (__any_sync(0xFFFFFFFFu, live && !isQ)) {
            float f[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) f[2 * i] = bf16_low(x[i]), f[2 * i + 1] = bf16_high(x[i]);
            float low = f[0], high = f[0];
            bool finite = true;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                low = fminf(low, f[i]);
                high = fmaxf(high, f[i]);
                finite &= fabsf(f[i]) < INFINITY;
            }
#pragma unroll
            for (int d = 1; d < 8; d <<= 1) {
                low = fminf(low, __shfl_xor_sync(0xFFFFFFFFu, low, d));
                high = fmaxf(high, __shfl_xor_sync(0xFFFFFFFFu, high, d));
                finite &= __shfl_xor_sync(0xFFFFFFFFu, (int)finite, d) != 0;
            }
            const uint32_t scaleBits = pack_bf16(__fdiv_rn(__fsub_rn(high, low), 15.0f), low);  // scale | bias
            const float scale = bf16_low(scaleBits);
            finite &= scale < INFINITY;
            const float inverse = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
            uint32_t word = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                // (a scale so small that its reciprocal overflows: 0 * inf stays below code 0, the rest is code 15)
                const float code = fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(f[i], low), inverse)), 0.0f), 15.0f);
                word |= (finite ? (uint32_t)code : 0u) << (4 * i);
            }
            if (live && !isQ && slot != FF_NO_SLOT) {
                if (slot < a.slotCount) {
                    const uint32_t inPage = slot & (a.page.pageTokens - 1u);
                    uint8_t *block = a.pages + (uint64_t)(slot >> a.pageShift) * a.page.pageBytes + (uint64_t)head * a.page.blockBytes + (isK ? 0u : a.page.values);
                    *reinterpret_cast<uint32_t *>(block + inPage * a.page.codeBytes + inHead * 4u) = word;
                    if ((inHead & 7u) == 0u)
                        *reinterpret_cast<uint32_t *>(block + a.page.keyWords + inPage * a.page.wordBytes + (inHead >> 3) * 4u) = finite ? scaleBits : 0x7FC07FC0u;
                } else if (inHead == 0u) {
                    *a.errorFlag = kFlagPage;
                }
            }
        }
    }
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
    a.headsPerUnit = perWarp;
    a.unitsPerToken = (heads + a.headsPerUnit - 1) / a.headsPerUnit;
    const uint64_t units = (uint64_t)tokens * a.unitsPerToken;
    const dim3 grid((uint32_t)((units + 3) / 4)), block(128);
    const bool interleaved = rope.layout == FF_ROPE_INTERLEAVED;
    cudaError_t st;
    if (cfg.headDim == 64) st = interleaved ? launch_pdl(k_rope_rows<64, true>, grid, block, 0, stream, a) : launch_pdl(k_rope_rows<64, false>, grid, block, 0, stream, a);
    else if (cfg.headDim == 128) st = interleaved ? launch_pdl(k_rope_rows<128, true>, grid, block, 0, stream, a) : launch_pdl(k_rope_rows<128, false>, grid, block, 0, stream, a);
    else st = interleaved ? launch_pdl(k_rope_rows<256, true>, grid, block, 0, stream, a) : launch_pdl(k_rope_rows<256, false>, grid, block, 0, stream, a);
    return launched(att, st, "k_rope_rows", error);
}

// ---- read-back ---------------------------------------------------------------------------------

struct ReadArgs {
    const uint8_t *pages;
    const uint32_t *slots;
    uint16_t *k, *v;
    uint32_t tokens, kvHeads, slotCount, pageShift, dim;
    PageLayout page;
    uint32_t *errorFlag;
};

// Eight values a thread.  Bound by the bytes written.
__global__ void __launch_bounds__(256) k_cache_read(const ReadArgs a) {
    pdl_enter();
    const uint32_t perHead = a.dim / 8, perRow = a.kvHeads * perHead, kinds = (a.k ? 1u : 0u) + (a.v ? 1u : 0u);
    const uint64_t total = (uint64_t)a.tokens * perRow * kinds;
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (uint64_t)gridDim.x * blockDim.x) {
        const uint32_t inRow = (uint32_t)(i % perRow);
        const uint64_t rest = i / perRow;
        const uint32_t token = (uint32_t)(rest / kinds);
        const bool key = a.k && rest % kinds == 0;
        const uint32_t head = inRow / perHead, at = inRow % perHead;
        const uint32_t slot = __ldg(a.slots + token);
        uint4 o = make_uint4(0u, 0u, 0u, 0u);
        if (slot < a.slotCount) {
            const uint32_t inPage = slot & (a.page.pageTokens - 1u);
            const uint8_t *block = a.pages + (uint64_t)(slot >> a.pageShift) * a.page.pageBytes + (uint64_t)head * a.page.blockBytes + (key ? 0u : a.page.values);
            const uint32_t w = *reinterpret_cast<const uint32_t *>(block + inPage * a.page.codeBytes + at * 4u);
            const uint32_t sb = *reinterpret_cast<const uint32_t *>(block + a.page.keyWords + inPage * a.page.wordBytes + (at >> 3) * 4u);
            const float scale = bf16_low(sb), bias = bf16_high(sb);
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = __fadd_rn(__fmul_rn((float)((w >> (4 * j)) & 15u), scale), bias);
            o = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
        } else if (slot != FF_NO_SLOT) {
            *a.errorFlag = kFlagPage;
        }
        uint16_t *out = key ? a.k : a.v;
        *reinterpret_cast<uint4 *>(out + ((uint64_t)token * perRow + inRow) * 8u) = o;
    }
}

bool launch_cache_read(FFAttention *att, const uint8_t *pages, uint32_t pageCount, const uint32_t *slots, uint32_t tokens, uint16_t *k,
                       uint16_t *v, cudaStream_t stream, const char **error) {
    if (tokens == 0 || (!k && !v)) return true;
    const FFAttentionConfig &cfg = att->cfg;
    ReadArgs a{pages, slots, k, v, tokens, cfg.kvHeads, pageCount * cfg.pageTokens, shift_of(cfg.pageTokens), cfg.headDim, page_layout(cfg), att->errorFlag};
    const uint64_t total = (uint64_t)tokens * cfg.kvHeads * (cfg.headDim / 8) * ((k ? 1 : 0) + (v ? 1 : 0));
    const uint32_t grid = (uint32_t)std::min<uint64_t>((total + 255) / 256, (uint64_t)att->smCount * 32);
    return launched(att, launch_pdl(k_cache_read, dim3(grid), dim3(256), 0, stream, a), "k_cache_read", error);
}

}  // namespace ff

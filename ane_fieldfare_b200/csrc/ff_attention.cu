// Attention over the paged INT4 key/value cache: the handle, the entry points' checks, the kernels.
#include <algorithm>
#include <string>

#include "ff_attention.cuh"

namespace ff {

constexpr uint32_t kBlockKeys = 64;
constexpr uint32_t kSharedLaunch = 200000;  // what the launches over prefixes take besides their tiles, 0.1 ns

bool launch_attend(FFAttention *att, const AttendArgs &a, cudaStream_t stream, const char **error) {
    // Columns of a key/value head: up to 16 as columns of mma.sync, which then take as long as the cache's bytes; more as rows of
    // tcgen05.mma.  us as columns / as rows: 16 columns of 128, 64 requests of up to 16384 keys 72 / 98; 32 of 128, 16 requests of
    // up to 3000 keys 28 / 28; 2 of 256 in a window of 1024 13 / 20; 4 of 256, 8000 keys 20 / 33; 32 of 256, 20000 keys 68 / 45.  At
    // 256 values a head, where more than 8 columns spill registers, 9 to 16 go the slower way (10, 8 x 4000 keys 59 / 54; 16, 8000 keys
    // 42 / 34, in a window of 1024 24 / 21): the boundary is one for all head sizes.
    if (a.maxRows * (a.heads / a.kvHeads) <= 16) return launch_attend_rows(att, a, stream, error);
    return launch_attend_tiles(att, a, stream, error);
}

// Whether groups share: their rows over their prefixes in one launch and the requests' rows from behind them in another, or the requests' launch
// alone, over all of their keys, where the other would take longer than it saves.  us alone / with both: 8 requests of 4 columns of
// 128 behind 4096 keys 17.8 / 25.8, 16384 42 / 34; 64 behind 1024 31 / 30, 4096 80 / 35, 16384 271 / 51; 16 of 8 rows of 2 of 256 behind
// 1024 48 / 43 (the rule takes the former), 4096 103 / 50, 16384 323 / 73; 16 of 8 rows of 7 of 64 behind 16384 49 / 47 (likewise).  It goes by
// what the host knows: all rows as if behind the longest prefix, every request as if it had as many of them.
static bool few_of_group(const FFAttentionConfig &c, uint32_t tokens) { return (uint64_t)tokens * (c.heads / c.kvHeads) <= (c.headDim == 256 ? 8 : 16); }
static bool few_of_request(const FFAttentionConfig &c, uint32_t maxRows) { return (uint64_t)maxRows * (c.heads / c.kvHeads) <= 16; }
bool attend_shares(const FFAttentionConfig &c, uint32_t tokens, uint32_t tableKeys, uint32_t requests, uint32_t maxRows, uint32_t groups, uint32_t maxPrefix) {
    if (!groups || maxPrefix == FF_SHARE_ALWAYS) return groups != 0;
    const uint32_t group = c.heads / c.kvHeads, dim = c.headDim, size = dim == 256 ? 2 : dim == 128 ? 1 : 0;
    const uint32_t active = std::min(requests, tokens), rows = active ? std::min(maxRows, (tokens + active - 1) / active) : 0;  // requests with rows, and theirs (as if all had as many)
    const bool fewOfRequest = few_of_request(c, maxRows), fewOfGroup = few_of_group(c, tokens);
    // what 64 keys cost a tile of columns, 0.1 ns of the whole GPU: of up to 4, 8 and 16, of 128 (where requests fill a part of them)
    static const uint32_t few[3][3] = {{14, 15, 20}, {20, 21, 35}, {37, 42, 90}}, many[3] = {40, 44, 63}, full[3] = {50, 62, 78};
    const uint64_t columns = (uint64_t)maxRows * group;
    const uint32_t of = columns <= 4 ? 0 : columns <= 8 ? 1 : 2, width = fewOfRequest ? 4u << of : kTileRows;
    auto tiles = [&](uint64_t n, uint32_t wide) {  // of n rows
        return group <= wide ? (n + wide / group - 1) / (wide / group) : n * ((group + wide - 1) / wide);
    };
    const uint64_t apart = active * tiles(rows, width) * (fewOfRequest ? few[size][of] : many[size]);
    const uint64_t together = std::max<uint64_t>(groups, fewOfGroup ? tiles(tokens, 16) : tiles(tokens, kTileRows)) * (fewOfGroup ? few[size][dim == 256 ? 1 : 2] : full[size]);
    const uint64_t keys = std::min(maxPrefix, tableKeys) / kBlockKeys;
    return apart > together && (apart - together) * keys * c.kvHeads > kSharedLaunch;
}

// Each launch goes to the kernel that its columns ask for, as in launch_attend; those of a group are all its rows' (bounded by the rows of the
// call; at 256 values a head eight, where more spill registers).
bool launch_attend_shared(FFAttention *att, const AttendArgs &a, cudaStream_t stream, const char **error) {
    AttendArgs b = a;
    b.maxRows = b.tokens;
    if (!(few_of_group(att->cfg, a.tokens) ? launch_attend_prefix_rows(att, b, stream, error) : launch_attend_prefix_tiles(att, b, stream, error))) return false;
    return few_of_request(att->cfg, a.maxRows) ? launch_attend_suffix_rows(att, a, stream, error) : launch_attend_suffix_tiles(att, a, stream, error);
}

}  // namespace ff

using namespace ff;

namespace {

bool supported(const FFAttentionConfig &c, const char **error) {
    if (c.kvHeads == 0 || c.heads == 0 || c.heads % c.kvHeads || c.heads / c.kvHeads > 64 || c.heads > 1024)
        return fail(error, "heads must be a multiple of kvHeads, up to 64 query heads a key/value head and 1024 in all");
    if (c.headDim != 64 && c.headDim != 128 && c.headDim != 256) return fail(error, "headDim must be 64, 128 or 256");
    if (c.pageTokens < 16 || c.pageTokens > 256 || (c.pageTokens & (c.pageTokens - 1)))
        return fail(error, "pageTokens must be 16, 32, 64, 128 or 256");
    if (c.maxRequests == 0 || c.maxTokens == 0 || c.maxRequests > (1u << 20) || c.maxTokens > (1u << 24))
        return fail(error, "need 1..2^20 requests and 1..2^24 rows");
    return true;
}

bool begin(FFAttention *att, const char **error) {
    if (error) *error = nullptr;
    if (!att) return fail(error, "null attention handle");
    FF_CUDA_OK(cudaSetDevice(att->device), error);
    return true;
}

bool aligned(const void *p, uint32_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1u)) == 0; }

// rows of `heads` heads: 16-byte pieces, and indexes that stay below 2^64
bool check_heads(const FFAttention *att, const void *x, uint32_t stride, uint32_t heads, const char *what, const char **error) {
    if (!x) return fail(error, std::string(what) + " pointer is null");
    if (stride < heads * att->cfg.headDim) return fail(error, std::string(what) + " row stride is too small");
    if (!aligned(x, 16) || stride % 8) return fail(error, std::string(what) + " rows must be 16-byte aligned (stride a multiple of 8 elements)");
    return true;
}

bool check_tokens(const FFAttention *att, uint32_t tokens, const char **error) {
    if (tokens > att->cfg.maxTokens)
        return fail(error, std::to_string(tokens) + " rows exceed the handle's maxTokens " + std::to_string(att->cfg.maxTokens));
    return true;
}

bool check_cache(const FFAttention *att, const void *pages, uint32_t pageCount, const char **error) {
    if (!pages) return fail(error, "pages pointer is null");
    if (!aligned(pages, 16)) return fail(error, "pages must be 16-byte aligned");
    if ((uint64_t)pageCount * att->cfg.pageTokens >= FF_NO_SLOT) return fail(error, "the cache has more slots than 32 bits name");
    return true;
}

bool check_requests(const FFAttention *att, uint32_t requests, const char **error) {
    if (requests > att->cfg.maxRequests)
        return fail(error, std::to_string(requests) + " requests exceed the handle's maxRequests " + std::to_string(att->cfg.maxRequests));
    return true;
}

// the block table, and `starts` (one per request, or one more) and lengths; without requests `starts` alone
bool check_table(const uint32_t *blockTable, uint32_t tableStride, const uint32_t *starts, const char *startsName, const uint32_t *lengths, uint32_t requests, const char **error) {
    if (!starts || !aligned(starts, 4)) return fail(error, std::string(startsName) + " must be non-null and 4-byte aligned");
    if (requests == 0) return true;
    if (!lengths || !aligned(lengths, 4)) return fail(error, "lengths must be non-null and 4-byte aligned");
    if (!blockTable || !aligned(blockTable, 4)) return fail(error, "blockTable must be non-null and 4-byte aligned");
    if (tableStride == 0) return fail(error, "tableStride must be positive");
    return true;
}

constexpr uint32_t kMostListed = 1u << 20;

// The workspace of ff_attention_shared: units in parts, the rows' maxima and sums, their values.
struct SharedLayout {
    uint64_t stats, values, bytes;
};
SharedLayout shared_layout(const FFAttentionConfig &c, uint32_t tokens) {
    const uint64_t rows = (uint64_t)tokens * c.heads;
    SharedLayout l{kSharedCtas * sizeof(uint4), 0, 0};
    l.values = (l.stats + rows * sizeof(float2) + 15) / 16 * 16;
    l.bytes = l.values + rows * c.headDim * sizeof(float);
    return l;
}

// keys that a row of the block table has room for
uint32_t table_keys(const FFAttentionConfig &c, uint32_t tableStride) { return (uint32_t)std::min<uint64_t>((uint64_t)tableStride * c.pageTokens, UINT32_MAX); }

bool check_rope(const FFAttention *att, const FFRope *rope, const uint32_t *positions, const char **error) {
    if (!rope) return fail(error, "rope is null");
    if (rope->rotaryDim % 16 || rope->rotaryDim > att->cfg.headDim) return fail(error, "rotaryDim must be a multiple of 16 up to headDim");
    if (rope->layout != FF_ROPE_HALVES && rope->layout != FF_ROPE_INTERLEAVED) return fail(error, "unknown rotary layout");
    if (rope->rotaryDim && (!rope->table || !aligned(rope->table, 16) || rope->positions == 0))
        return fail(error, "the rotary table must be non-null, 16-byte aligned and hold a position");
    if (rope->rotaryDim && (!positions || !aligned(positions, 4))) return fail(error, "positions must be non-null and 4-byte aligned");
    return true;
}

}  // namespace

extern "C" {

uint64_t ff_cache_page_bytes(const FFAttentionConfig *config) {
    return config && supported(*config, nullptr) ? page_layout(*config).pageBytes : 0;
}

void ff_attention_destroy(FFAttention *att) {
    if (!att) return;
    cudaSetDevice(att->device);
    cudaDeviceSynchronize();
    cudaFree(att->errorFlag);
    cudaFree(att->planCount);
    cudaFree(att->partials);
    cudaFree(att->stats);
    cudaFree(att->arrived);
    delete att;
}

FFAttention *ff_attention_create(int32_t deviceOrdinal, const FFAttentionConfig *config, const char **error) {
    if (error) *error = nullptr;
    if (!config) {
        fail(error, "config is null");
        return nullptr;
    }
    if (!supported(*config, error)) return nullptr;
    int count = 0;
    cudaError_t st = cudaGetDeviceCount(&count);
    if (st != cudaSuccess || count == 0) {
        fail(error, std::string("no CUDA device: ") + (st != cudaSuccess ? cudaGetErrorString(st) : "device count is 0"));
        return nullptr;
    }
    if (deviceOrdinal < 0 || deviceOrdinal >= count) {
        fail(error, "device ordinal " + std::to_string(deviceOrdinal) + " out of range");
        return nullptr;
    }
    cudaDeviceProp prop{};
    if ((st = cudaSetDevice(deviceOrdinal)) != cudaSuccess || (st = cudaGetDeviceProperties(&prop, deviceOrdinal)) != cudaSuccess) {
        fail(error, std::string("device: ") + cudaGetErrorString(st));
        return nullptr;
    }
    if (prop.major != 10) {
        fail(error, "this library is built for sm_100a only; device is sm_" + std::to_string(prop.major) + std::to_string(prop.minor));
        return nullptr;
    }
    FFAttention *att = new FFAttention();
    att->device = deviceOrdinal;
    att->smCount = prop.multiProcessorCount;
    att->cfg = *config;
    auto alloc = [&](auto **p, size_t n) {
        if (st != cudaSuccess) return;
        const size_t bytes = std::max<size_t>(n, 1) * sizeof(**p);
        st = cudaMalloc(reinterpret_cast<void **>(p), bytes);
        if (st == cudaSuccess) st = cudaMemset(*p, 0, bytes);
        att->scratchBytes += bytes;
    };
    alloc(&att->errorFlag, 1);
    alloc(&att->planCount, 1);
    att->rowsCtas = attend_rows_ctas(att->smCount);
    alloc(&att->partials, 2 * std::max((size_t)att->rowsCtas * kPartialValues, (size_t)att->smCount * kTileRows * config->headDim));
    alloc(&att->stats, 2 * std::max((size_t)att->rowsCtas * kPartialColumns, (size_t)att->smCount * kTileRows));
    alloc(&att->arrived, 3 * att->rowsCtas);
    if (st == cudaSuccess) st = cudaDeviceSynchronize();
    if (st != cudaSuccess) {
        fail(error, std::string("attention scratch: ") + cudaGetErrorString(st));
        ff_attention_destroy(att);
        return nullptr;
    }
    return att;
}

FFAttentionInfo ff_attention_get_info(const FFAttention *att) {
    FFAttentionInfo info{};
    if (!att) return info;
    info.kernelLaunches = att->kernelLaunches;
    info.scratchBytes = att->scratchBytes;
    info.deviceOrdinal = (uint32_t)att->device;
    info.smCount = (uint32_t)att->smCount;
    cudaSetDevice(att->device);
    cudaMemcpy(&info.deviceErrorFlag, att->errorFlag, sizeof(uint32_t), cudaMemcpyDeviceToHost);
    return info;
}

bool ff_attention_reset_device_error(FFAttention *att, const char **error) {
    if (!begin(att, error)) return false;
    FF_CUDA_OK(cudaDeviceSynchronize(), error);
    // a call that gave up a wait (flag 17) leaves counts behind; the next one would join parts that are not there yet
    FF_CUDA_OK(cudaMemset(att->arrived, 0, 3 * att->rowsCtas * sizeof(uint32_t)), error);
    FF_CUDA_OK(cudaMemset(att->planCount, 0, sizeof(uint32_t)), error);
    FF_CUDA_OK(cudaMemset(att->errorFlag, 0, sizeof(uint32_t)), error);
    FF_CUDA_OK(cudaDeviceSynchronize(), error);  // (a memset may return before it is done; other streams do not wait for it)
    return true;
}

bool ff_cache_plan_shared(FFAttention *att, const uint32_t *oldLengths, const uint32_t *newLengths, uint32_t requests, uint32_t *blockTable,
                          uint32_t tableStride, uint32_t *freePages, uint32_t pageCount, const uint32_t *freeCountIn, uint32_t *freeCountOut,
                          uint32_t *rowStart, uint32_t *positions, uint32_t *slots, uint32_t rows, const uint32_t *heldPages, void *stream, const char **error) {
    if (!begin(att, error)) return false;
    if (requests > att->cfg.maxRequests)
        return fail(error, std::to_string(requests) + " requests exceed the handle's maxRequests " + std::to_string(att->cfg.maxRequests));
    if (!check_tokens(att, rows, error)) return false;
    if (!oldLengths || !newLengths || !blockTable || !freePages || !freeCountIn || !freeCountOut || !rowStart || (rows && (!positions || !slots)))
        return fail(error, "null argument");
    const uintptr_t all = reinterpret_cast<uintptr_t>(oldLengths) | reinterpret_cast<uintptr_t>(newLengths) | reinterpret_cast<uintptr_t>(blockTable) |
                          reinterpret_cast<uintptr_t>(freePages) | reinterpret_cast<uintptr_t>(freeCountIn) | reinterpret_cast<uintptr_t>(freeCountOut) |
                          reinterpret_cast<uintptr_t>(rowStart) | reinterpret_cast<uintptr_t>(positions) | reinterpret_cast<uintptr_t>(slots) |
                          reinterpret_cast<uintptr_t>(heldPages);
    if (all & 3u) return fail(error, "arrays must be 4-byte aligned");
    if (tableStride == 0) return fail(error, "tableStride must be positive");
    if ((uint64_t)requests * tableStride > 1u << 30) return fail(error, "the block table has more than 2^30 entries");
    if ((uint64_t)pageCount * att->cfg.pageTokens >= FF_NO_SLOT) return fail(error, "the cache has more slots than 32 bits name");
    return launch_cache_plan(att, oldLengths, newLengths, requests, blockTable, tableStride, freePages, pageCount, freeCountIn, freeCountOut,
                             rowStart, positions, slots, rows, heldPages, static_cast<cudaStream_t>(stream), error);
}

bool ff_cache_plan(FFAttention *att, const uint32_t *oldLengths, const uint32_t *newLengths, uint32_t requests, uint32_t *blockTable,
                   uint32_t tableStride, uint32_t *freePages, uint32_t pageCount, const uint32_t *freeCountIn, uint32_t *freeCountOut,
                   uint32_t *rowStart, uint32_t *positions, uint32_t *slots, uint32_t rows, void *stream, const char **error) {
    return ff_cache_plan_shared(att, oldLengths, newLengths, requests, blockTable, tableStride, freePages, pageCount, freeCountIn, freeCountOut, rowStart,
                                positions, slots, rows, nullptr, stream, error);
}

bool ff_rope_table(FFAttention *att, const FFRopeConfig *config, float *table, uint32_t positions, void *stream, const char **error) {
    if (!begin(att, error)) return false;
    if (!config || !table) return fail(error, "null argument");
    if (!aligned(table, 16)) return fail(error, "the rotary table must be 16-byte aligned");
    if (config->rotaryDim % 16 || config->rotaryDim > att->cfg.headDim) return fail(error, "rotaryDim must be a multiple of 16 up to headDim");
    if (!(config->base > 0.0)) return fail(error, "base must be positive");
    if (config->scaling > FF_ROPE_BY_PARTS) return fail(error, "unknown rotary scaling");
    if (config->scaling != FF_ROPE_PLAIN && !(config->factor > 0.0)) return fail(error, "factor must be positive");
    if (config->scaling == FF_ROPE_BY_PARTS && !(config->highTurns > config->lowTurns && config->originalContext > 0.0))
        return fail(error, "scaling by parts needs highTurns above lowTurns and an original context");
    return launch_rope_table(att, *config, table, positions, static_cast<cudaStream_t>(stream), error);
}

bool ff_rope(FFAttention *att, const uint16_t *x, uint32_t xStride, const FFRope *rope, const uint32_t *positions, uint32_t heads, uint32_t tokens,
             uint16_t *y, uint32_t yStride, void *stream, const char **error) {
    if (!begin(att, error)) return false;
    if (heads == 0 || heads > 1024) return fail(error, "need 1..1024 heads");
    if (tokens == 0) return true;
    if (!check_tokens(att, tokens, error) || !check_heads(att, x, xStride, heads, "input", error) ||
        !check_heads(att, y, yStride, heads, "output", error) || !check_rope(att, rope, positions, error))
        return false;
    RopeRows rows{};
    rows.q = x;
    rows.qStride = xStride;
    rows.qHeads = heads;
    rows.qOut = y;
    rows.qOutStride = yStride;
    return launch_rope_rows(att, rows, *rope, positions, nullptr, tokens, nullptr, 0, static_cast<cudaStream_t>(stream), error);
}

bool ff_cache_append(FFAttention *att, const uint16_t *q, uint32_t qStride, const uint16_t *k, uint32_t kStride, const uint16_t *v,
                     uint32_t vStride, const FFRope *rope, const uint32_t *positions, const uint32_t *slots, uint32_t tokens, uint16_t *qOut,
                     uint32_t qOutStride, void *pages, uint32_t pageCount, void *stream, const char **error) {
    if (!begin(att, error)) return false;
    const FFAttentionConfig &c = att->cfg;
    if (tokens == 0) return true;
    if (!check_tokens(att, tokens, error) || !check_heads(att, k, kStride, c.kvHeads, "key", error) ||
        !check_heads(att, v, vStride, c.kvHeads, "value", error) || !check_rope(att, rope, positions, error) ||
        !check_cache(att, pages, pageCount, error))
        return false;
    if (q && (!check_heads(att, q, qStride, c.heads, "query", error) || !check_heads(att, qOut, qOutStride, c.heads, "query output", error)))
        return false;
    if (!slots || !aligned(slots, 4)) return fail(error, "slots must be non-null and 4-byte aligned");
    RopeRows rows{q, k, v, qStride, kStride, vStride, c.heads, qOut, qOutStride};
    return launch_rope_rows(att, rows, *rope, positions, slots, tokens, static_cast<uint8_t *>(pages), pageCount, static_cast<cudaStream_t>(stream), error);
}

bool ff_cache_read(FFAttention *att, const void *pages, uint32_t pageCount, const uint32_t *slots, uint32_t tokens, uint16_t *k, uint16_t *v,
                   void *stream, const char **error) {
    if (!begin(att, error)) return false;
    if (tokens == 0) return true;
    if (!check_tokens(att, tokens, error) || !check_cache(att, pages, pageCount, error)) return false;
    if (!slots || !aligned(slots, 4)) return fail(error, "slots must be non-null and 4-byte aligned");
    if (!aligned(k, 16) || !aligned(v, 16)) return fail(error, "output rows must be 16-byte aligned");
    return launch_cache_read(att, static_cast<const uint8_t *>(pages), pageCount, slots, tokens, k, v, static_cast<cudaStream_t>(stream), error);
}

bool ff_attention(FFAttention *att, const uint16_t *q, uint32_t qStride, uint32_t tokens, const void *pages, uint32_t pageCount,
                  const uint32_t *blockTable, uint32_t tableStride, const uint32_t *rowStart, const uint32_t *lengths, uint32_t requests,
                  uint32_t maxRows, float scale, uint32_t window, uint32_t sinks, uint16_t *out, uint32_t outStride, void *stream,
                  const char **error) {
    if (!begin(att, error)) return false;
    const FFAttentionConfig &c = att->cfg;
    if (tokens == 0) return true;
    if (!check_tokens(att, tokens, error) || !check_heads(att, q, qStride, c.heads, "query", error) ||
        !check_heads(att, out, outStride, c.heads, "output", error) || !check_cache(att, pages, pageCount, error))
        return false;
    if (requests > c.maxRequests)
        return fail(error, std::to_string(requests) + " requests exceed the handle's maxRequests " + std::to_string(c.maxRequests));
    if (!blockTable || !rowStart || !lengths) return fail(error, "null argument");
    if (!aligned(blockTable, 4) || !aligned(rowStart, 4) || !aligned(lengths, 4)) return fail(error, "arrays must be 4-byte aligned");
    if (tableStride == 0 || maxRows == 0) return fail(error, "tableStride and maxRows must be positive");
    if (!(scale > 0.0f && scale < INFINITY)) return fail(error, "scale must be positive and finite");
    if (sinks && !window) return fail(error, "sinks need a window");
    AttendArgs a{q, out, qStride, outStride, tokens, static_cast<const uint8_t *>(pages), pageCount, tableStride, table_keys(c, tableStride), blockTable, rowStart, lengths, requests,
                 std::min(maxRows, std::max(1u, tokens)), scale, window, sinks, c.heads, c.kvHeads, page_layout(c), att->errorFlag, nullptr, 0, {}};
    return launch_attend(att, a, static_cast<cudaStream_t>(stream), error);
}

bool ff_block_means(FFAttention *att, const void *pages, uint32_t pageCount, const uint32_t *blockTable, uint32_t tableStride, const uint32_t *oldLengths,
                    const uint32_t *newLengths, uint32_t requests, uint16_t *means, void *stream, const char **error) {
    if (!begin(att, error)) return false;
    const FFAttentionConfig &c = att->cfg;
    if (!check_requests(att, requests, error)) return false;
    if (requests == 0) return true;
    if (!check_cache(att, pages, pageCount, error) || !check_table(blockTable, tableStride, oldLengths, "oldLengths", newLengths, requests, error)) return false;
    if (!means || !aligned(means, 16)) return fail(error, "means must be non-null and 16-byte aligned");
    return launch_block_means(att, static_cast<const uint8_t *>(pages), pageCount, blockTable, tableStride, table_keys(c, tableStride), oldLengths, newLengths,
                              requests, means, static_cast<cudaStream_t>(stream), error);
}

bool ff_select_blocks(FFAttention *att, const uint16_t *q, uint32_t qStride, uint32_t tokens, const uint16_t *means, uint32_t pageCount,
                      const uint32_t *blockTable, uint32_t tableStride, const uint32_t *rowStart, const uint32_t *lengths, uint32_t requests,
                      uint32_t blocks, uint32_t first, uint32_t last, uint32_t *ids, void *stream, const char **error) {
    if (!begin(att, error)) return false;
    const FFAttentionConfig &c = att->cfg;
    if (blocks == 0 || blocks > kMostListed) return fail(error, "need 1..2^20 blocks a list");
    if (last == 0) return fail(error, "a row's own block is always in its list: last must be positive");
    if (first > blocks || last > blocks - first) return fail(error, "the first and the last blocks are more than a list holds");
    if (tokens == 0) return true;
    if (!check_tokens(att, tokens, error) || !check_heads(att, q, qStride, c.heads, "query", error) || !check_requests(att, requests, error) ||
        !check_table(blockTable, tableStride, rowStart, "rowStart", lengths, requests, error))
        return false;
    if (!means || !aligned(means, 16)) return fail(error, "means must be non-null and 16-byte aligned");
    if (!ids || !aligned(ids, 4)) return fail(error, "ids must be non-null and 4-byte aligned");
    if ((uint64_t)pageCount * c.pageTokens >= FF_NO_SLOT) return fail(error, "the cache has more slots than 32 bits name");
    const uint64_t keys = (uint64_t)tableStride * c.pageTokens;
    if (keys > 1u << 21) return fail(error, "block table rows of more than 2^21 keys: their scores do not fit a CTA");
    return launch_select_blocks(att, q, qStride, tokens, means, pageCount, blockTable, tableStride, (uint32_t)((keys + kBlockKeys - 1) / kBlockKeys), rowStart,
                                lengths, requests, blocks, first, last, ids, static_cast<cudaStream_t>(stream), error);
}

bool ff_attention_selected(FFAttention *att, const uint16_t *q, uint32_t qStride, uint32_t tokens, const void *pages, uint32_t pageCount,
                           const uint32_t *blockTable, uint32_t tableStride, const uint32_t *rowStart, const uint32_t *lengths, uint32_t requests,
                           const uint32_t *ids, uint32_t blocks, float scale, uint16_t *out, uint32_t outStride, void *stream, const char **error) {
    if (!begin(att, error)) return false;
    const FFAttentionConfig &c = att->cfg;
    if (blocks == 0 || blocks > kMostListed) return fail(error, "need 1..2^20 blocks a list");
    if (!(scale > 0.0f && scale < INFINITY)) return fail(error, "scale must be positive and finite");
    if (tokens == 0) return true;
    if (!check_tokens(att, tokens, error) || !check_heads(att, q, qStride, c.heads, "query", error) ||
        !check_heads(att, out, outStride, c.heads, "output", error) || !check_cache(att, pages, pageCount, error) ||
        !check_requests(att, requests, error) || !check_table(blockTable, tableStride, rowStart, "rowStart", lengths, requests, error))
        return false;
    if (!ids || !aligned(ids, 4)) return fail(error, "ids must be non-null and 4-byte aligned");
    AttendArgs a{q, out, qStride, outStride, tokens, static_cast<const uint8_t *>(pages), pageCount, tableStride, table_keys(c, tableStride), blockTable,
                 rowStart, lengths, requests, 1, scale, 0, 0, c.heads, c.kvHeads, page_layout(c), att->errorFlag, ids, blocks, {}};
    return launch_attend_listed(att, a, static_cast<cudaStream_t>(stream), error);
}

uint64_t ff_attention_shared_bytes(const FFAttentionConfig *config, uint32_t tokens) {
    return config && supported(*config, nullptr) ? shared_layout(*config, tokens).bytes : 0;
}

bool ff_attention_shares(const FFAttentionConfig *config, uint32_t tokens, uint32_t tableStride, uint32_t requests, uint32_t maxRows, uint32_t groups, uint32_t maxPrefix) {
    return config && supported(*config, nullptr) && attend_shares(*config, tokens, table_keys(*config, tableStride), requests, std::min(maxRows, tokens), groups, maxPrefix);
}

bool ff_attention_shared(FFAttention *att, const uint16_t *q, uint32_t qStride, uint32_t tokens, const void *pages, uint32_t pageCount,
                         const uint32_t *blockTable, uint32_t tableStride, const uint32_t *rowStart, const uint32_t *lengths, uint32_t requests,
                         uint32_t maxRows, const uint32_t *groupStart, const uint32_t *prefixLengths, uint32_t groups, uint32_t maxPrefix, float scale, void *workspace,
                         uint16_t *out, uint32_t outStride, void *stream, const char **error) {
    if (!begin(att, error)) return false;
    const FFAttentionConfig &c = att->cfg;
    if (!(scale > 0.0f && scale < INFINITY)) return fail(error, "scale must be positive and finite");
    if (tokens == 0) return true;
    if (maxRows == 0) return fail(error, "maxRows must be positive");
    if (!check_tokens(att, tokens, error) || !check_heads(att, q, qStride, c.heads, "query", error) ||
        !check_heads(att, out, outStride, c.heads, "output", error) || !check_cache(att, pages, pageCount, error) ||
        !check_requests(att, requests, error) || !check_table(blockTable, tableStride, rowStart, "rowStart", lengths, requests, error))
        return false;
    if (groups > requests) return fail(error, "more groups than requests");
    if (groups && (!groupStart || !prefixLengths || !aligned(groupStart, 4) || !aligned(prefixLengths, 4)))
        return fail(error, "groupStart and prefixLengths must be non-null and 4-byte aligned");
    const bool shares = attend_shares(c, tokens, table_keys(c, tableStride), requests, std::min(maxRows, tokens), groups, maxPrefix);
    if (shares && (!workspace || !aligned(workspace, 16))) return fail(error, "workspace must be non-null and 16-byte aligned");
    const SharedLayout l = shared_layout(c, tokens);
    uint8_t *w = static_cast<uint8_t *>(workspace);
    AttendArgs a{q, out, qStride, outStride, tokens, static_cast<const uint8_t *>(pages), pageCount, tableStride, table_keys(c, tableStride), blockTable,
                 rowStart, lengths, requests, std::min(maxRows, tokens), scale, 0, 0, c.heads, c.kvHeads, page_layout(c), att->errorFlag, nullptr, 0,
                 {groupStart, prefixLengths, groups, reinterpret_cast<uint4 *>(w), reinterpret_cast<float2 *>(w + l.stats), reinterpret_cast<float *>(w + l.values)}};
    if (!shares) return launch_attend(att, a, static_cast<cudaStream_t>(stream), error);
    if (att->smCount > (int)kSharedCtas) return fail(error, "more SMs than the workspace has room for");
    return launch_attend_shared(att, a, static_cast<cudaStream_t>(stream), error);
}

}  // extern "C"

// Attention over the paged INT4 key/value cache: the handle, the entry points' checks, the kernels.
#include <algorithm>
#include <string>

#include "ff_attention.cuh"

namespace ff {

bool launch_attend(FFAttention *att, const AttendArgs &a, cudaStream_t stream, const char **error) {
    // Columns of a key/value head: up to 16 as columns of mma.sync, which then take as long as the cache's bytes; more as rows of
    // tcgen05.mma.  us as columns / as rows: 16 columns of 128, 64 requests of up to 16384 keys 72 / 98; 32 of 128, 16 requests of
    // up to 3000 keys 28 / 28; 2 of 256 in a window of 1024 13 / 20; 4 of 256, 8000 keys 20 / 33; 32 of 256, 20000 keys 68 / 45.  At
    // 256 values a head, where more than 8 columns spill registers, 9 to 16 go the slower way (10, 8 x 4000 keys 59 / 54; 16, 8000 keys
    // 42 / 34, in a window of 1024 24 / 21): the boundary is one for all head sizes.
    if (a.maxRows * (a.heads / a.kvHeads) <= 16) return launch_attend_rows(att, a, stream, error);
    return launch_attend_tiles(att, a, stream, error);
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

bool ff_cache_plan(FFAttention *att, const uint32_t *oldLengths, const uint32_t *newLengths, uint32_t requests, uint32_t *blockTable,
                   uint32_t tableStride, uint32_t *freePages, uint32_t pageCount, const uint32_t *freeCountIn, uint32_t *freeCountOut,
                   uint32_t *rowStart, uint32_t *positions, uint32_t *slots, uint32_t rows, void *stream, const char **error) {
    if (!begin(att, error)) return false;
    if (requests > att->cfg.maxRequests)
        return fail(error, std::to_string(requests) + " requests exceed the handle's maxRequests " + std::to_string(att->cfg.maxRequests));
    if (!check_tokens(att, rows, error)) return false;
    if (!oldLengths || !newLengths || !blockTable || !freePages || !freeCountIn || !freeCountOut || !rowStart || (rows && (!positions || !slots)))
        return fail(error, "null argument");
    const uintptr_t all = reinterpret_cast<uintptr_t>(oldLengths) | reinterpret_cast<uintptr_t>(newLengths) | reinterpret_cast<uintptr_t>(blockTable) |
                          reinterpret_cast<uintptr_t>(freePages) | reinterpret_cast<uintptr_t>(freeCountIn) | reinterpret_cast<uintptr_t>(freeCountOut) |
                          reinterpret_cast<uintptr_t>(rowStart) | reinterpret_cast<uintptr_t>(positions) | reinterpret_cast<uintptr_t>(slots);
    if (all & 3u) return fail(error, "arrays must be 4-byte aligned");
    if (tableStride == 0) return fail(error, "tableStride must be positive");
    if ((uint64_t)requests * tableStride > 1u << 30) return fail(error, "the block table has more than 2^30 entries");
    if ((uint64_t)pageCount * att->cfg.pageTokens >= FF_NO_SLOT) return fail(error, "the cache has more slots than 32 bits name");
    return launch_cache_plan(att, oldLengths, newLengths, requests, blockTable, tableStride, freePages, pageCount, freeCountIn, freeCountOut,
                             rowStart, positions, slots, rows, static_cast<cudaStream_t>(stream), error);
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
    AttendArgs a{q, out, qStride, outStride, tokens, static_cast<const uint8_t *>(pages), pageCount, tableStride,
                 (uint32_t)std::min<uint64_t>((uint64_t)tableStride * c.pageTokens, UINT32_MAX), blockTable, rowStart, lengths, requests,
                 std::min(maxRows, std::max(1u, tokens)), scale, window, sinks, c.heads, c.kvHeads, page_layout(c), att->errorFlag};
    return launch_attend(att, a, static_cast<cudaStream_t>(stream), error);
}

}  // extern "C"

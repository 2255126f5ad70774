// What the kernels of the INT4 key/value cache and its attention share: the handle, a page's layout, launches.
#pragma once

#include "ff_internal.cuh"

struct FFAttention {
    int device = 0;
    int smCount = 0;
    FFAttentionConfig cfg{};
    uint32_t *errorFlag = nullptr;  // device: one of the AttentionFlag values
    uint32_t *planCount = nullptr;  // device: CTAs of ff_cache_plan that are done (zero between launches)
    uint32_t rowsCtas = 0;          // CTAs that the scratch below serves
    float *partials = nullptr;      // device: outputs of units that several CTAs share, two parts a CTA
    float4 *stats = nullptr;        // device: their maxima and sums
    uint32_t *arrived = nullptr;    // device: parts of a shared unit that are there (zero between launches)
    uint64_t kernelLaunches = 0;
    uint64_t scratchBytes = 0;
};

namespace ff {

enum AttentionFlag : uint32_t {
    kFlagNoPage = 13,
    kFlagTableRow = 14,
    kFlagRows = 15,
    kFlagPage = 16,
    kFlagWait = 17,
    kFlagPosition = 18,
    kFlagWork = 19,
};

// A block: one key/value head of one page.  Offsets in bytes from its start.
struct PageLayout {
    uint32_t pageTokens, codeBytes, wordBytes;  // of a token's key (or value) of one head
    uint32_t keyWords, values, valueWords;      // where they begin; the key codes begin at 0
    uint32_t blockBytes;
    uint64_t pageBytes;
};
inline PageLayout page_layout(const FFAttentionConfig &c) {
    PageLayout l{};
    l.pageTokens = c.pageTokens;
    l.codeBytes = c.headDim / 2;
    l.wordBytes = c.headDim / kGroup * 4;
    l.keyWords = l.pageTokens * l.codeBytes;
    l.values = l.keyWords + l.pageTokens * l.wordBytes;
    l.valueWords = l.values + l.pageTokens * l.codeBytes;
    l.blockBytes = 2 * l.values;
    l.pageBytes = (uint64_t)l.blockBytes * c.kvHeads;
    return l;
}

// Partial results of units that several CTAs share: columns (rows times query heads of a key/value head) of a unit, and
// their output values, where requests have few rows (two CTAs an SM) and many (one).
constexpr uint32_t kPartialColumns = 16, kPartialValues = 4096, kTileRows = 128;

// Counts a launch and reports what it says.
inline bool launched(FFAttention *att, cudaError_t status, const char *what, const char **error) {
    if (status == cudaSuccess) status = cudaGetLastError();
    if (status != cudaSuccess) return fail(error, std::string(what) + ": " + cudaGetErrorString(status));
    att->kernelLaunches++;
    return true;
}

struct AttendArgs {
    const uint16_t *q;
    uint16_t *out;
    uint32_t qStride, outStride, tokens;
    const uint8_t *pages;
    uint32_t pageCount, tableStride, tableKeys;  // tableKeys: those that a row of the block table has room for
    const uint32_t *blockTable, *rowStart, *lengths;
    uint32_t requests, maxRows;
    float scale;
    uint32_t window, sinks;
    uint32_t heads, kvHeads;
    PageLayout page;
    uint32_t *errorFlag;
};

// ff_cache.cu
bool launch_cache_plan(FFAttention *att, const uint32_t *oldLengths, const uint32_t *newLengths, uint32_t requests, uint32_t *blockTable,
                       uint32_t tableStride, uint32_t *freePages, uint32_t pageCount, const uint32_t *freeCountIn, uint32_t *freeCountOut,
                       uint32_t *rowStart, uint32_t *positions, uint32_t *slots, uint32_t rows, cudaStream_t stream, const char **error);
bool launch_rope_table(FFAttention *att, const FFRopeConfig &config, float *table, uint32_t positions, cudaStream_t stream, const char **error);
// Rows of heads that a launch rotates (keys: also quantizes); null pointers: none.
struct RopeRows {
    const uint16_t *q, *k, *v;
    uint32_t qStride, kStride, vStride, qHeads;
    uint16_t *qOut;
    uint32_t qOutStride;
};
bool launch_rope_rows(FFAttention *att, const RopeRows &rows, const FFRope &rope, const uint32_t *positions, const uint32_t *slots,
                      uint32_t tokens, uint8_t *pages, uint32_t pageCount, cudaStream_t stream, const char **error);
bool launch_cache_read(FFAttention *att, const uint8_t *pages, uint32_t pageCount, const uint32_t *slots, uint32_t tokens, uint16_t *k,
                       uint16_t *v, cudaStream_t stream, const char **error);

// ff_attend_rows.cu
uint32_t attend_rows_ctas(int smCount);
bool launch_attend_rows(FFAttention *att, const AttendArgs &args, cudaStream_t stream, const char **error);

// ff_attend_tiles.cu
bool launch_attend_tiles(FFAttention *att, const AttendArgs &args, cudaStream_t stream, const char **error);

// ff_attention.cu
bool launch_attend(FFAttention *att, const AttendArgs &args, cudaStream_t stream, const char **error);

}  // namespace ff

// Device helpers of the two attention kernels over the paged INT4 cache.
#pragma once

#include <cuda_fp16.h>

#include "ff_attention.cuh"
#include "ff_mma_device.cuh"

namespace ff {

constexpr float kLazy = 8.0f;  // log2 by which a logit may pass the running maximum before outputs are rescaled
constexpr float kNone = -1e30f;  // the maximum of no logit: any is above it, and 2^(it - any) is 0
constexpr uint32_t kTileKeys = 64;

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ void sts64(uint32_t a, uint32_t x, uint32_t y) { asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(a), "r"(x), "r"(y) : "memory"); }
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// the NG scale words of a key
template <int NG>
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t (&w)[NG]) {
    if (NG == 4) asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1 % NG]), "=r"(w[2 % NG]), "=r"(w[3 % NG]) : "r"(a));
    else if (NG == 2) asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1 % NG]) : "r"(a));
    else w[0] = lds32(a);
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float low16(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high16(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
// 2^e, 0 below the normal numbers
__device__ __forceinline__ float power_of_two(int e) { return e < -126 ? 0.0f : __uint_as_float((uint32_t)(min(e, 127) + 127) << 23); }
// The factor from a product's units to logits: scale, log2 e and 2^e.  Never 0, which times the -infinity of a key that is not seen would be
// no number: below the smallest number all logits are 0 as far as 32 bits go.
__device__ __forceinline__ float logit_factor(float scale, int e) {
    const int half = e >> 1;
    return fmaxf(scale * 1.4426950408889634f * power_of_two(half) * power_of_two(e - half), 0x1p-149f);
}
// a scale word whose scale or bias is no number: its group of values stands for NaN
__device__ __forceinline__ bool is_broken(uint32_t w) { return (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u; }
// exponent field of the larger of 16 scale and |bias|
__device__ __forceinline__ uint32_t word_exponent(uint32_t w) { return max(((w & 0x7FFFu) >> 7) + 4u, (w & 0x7FFF0000u) >> 23); }
// 16-byte chunks of a key's codes in a tile are exchanged by the key's place: the tensor map's swizzle (128-, 64- or
// 32-byte rows)
template <int DIM>
__device__ __forceinline__ uint32_t chunk_flip(uint32_t key) {
    return DIM == 256 ? (key & 7u) << 4 : DIM == 128 ? ((key >> 1) & 3u) << 4 : ((key >> 2) & 1u) << 4;
}

// Work is counted in tiles, in 32 bits; what does not fit (seconds of the GPU's time) stays at the largest number, kTooMuch.
constexpr uint32_t kTooMuch = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t add_work(uint32_t a, uint32_t b) { return a + b < a ? kTooMuch : a + b; }
__device__ __forceinline__ uint32_t work_of(uint32_t tiles, uint32_t units) { return __umulhi(tiles, units) ? kTooMuch : tiles * units; }

// The cache's pages as tensors: codes [blocks][keys, values][tokens][bytes], a box the part of a tile that lies on one page, of
// `sides` of the two; scale words [blocks][keys, values][words], a box both sides of such a part.
bool make_pages_maps(CUtensorMap *codes, CUtensorMap *words, const AttendArgs &a, uint32_t dim, uint32_t sides, const char **error);

}  // namespace ff

// mxkv.cuh -- the MX-quantised paged KV cache: device view, row layout and the
// host-side checks its entry points share.
#pragma once

#include "common.cuh"

namespace fp4x {
namespace mxkv {

enum : uint32_t { FMT_FP8 = FP4X_MXFP8, FMT_FP4 = FP4X_MXFP4 };

// Device view of a cache.  Offsets into it are 64-bit (a pool of long contexts passes
// 4 GB), those within a page 32-bit: one widening multiply-add makes an address.
struct Cache {
    uint8_t *k, *ks, *v, *vs;
    uint32_t page_stride, scale_stride;  // bytes between pages
    uint32_t n_pages, page_shift, n_kv;
};

// Bytes of one row's codes, and its 32-blocks.
template <uint32_t FMT, uint32_t HD>
struct Row {
    static constexpr uint32_t NB = HD / 32;
    static constexpr uint32_t BYTES = FMT == FMT_FP8 ? HD : HD / 2;
    static constexpr uint32_t CHUNK = BYTES / 8;  // codes of the four dimensions 4g..4g+3 of every block
};

// Byte offsets of (page, head, row in page).
template <uint32_t FMT, uint32_t HD>
__device__ __forceinline__ uint64_t code_off(const Cache &c, uint32_t page, uint32_t head, uint32_t row) {
    return (uint64_t)page * c.page_stride + ((head << c.page_shift) + row) * Row<FMT, HD>::BYTES;
}
template <uint32_t HD>
__device__ __forceinline__ uint64_t scale_off(const Cache &c, uint32_t page, uint32_t head, uint32_t row) {
    return (uint64_t)page * c.scale_stride + ((head << c.page_shift) + row) * (HD / 32);
}

// Checks `c` and fills the device view; a message and false if it is not valid.
bool view(const char *who, const fp4x_mxkv *c, Cache &out);

inline bool aligned(const void *p, uint32_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace mxkv
}  // namespace fp4x

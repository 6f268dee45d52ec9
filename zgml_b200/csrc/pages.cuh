// Pages of a cache in 8 bits (PAGE_APPEND, PAGED_ATTENTION, PAGE_READ, PAGE_COPY; layout in include/zgml_cuda.h) as the kernels address them.
// A page holds `page` tokens (16, 32 or 64) of every key head, a head after the other: two scales and two words beside them, then keys, then values.  A value is a code, a whole
// number of -127 to 127, times its scale, a power of two; stored is code + 128.  Keys lie in tiles of 8 tokens by 32
// values and values in tiles of 16 tokens by 16 values, so that the 8 bytes at 8 * lane of a tile are what lane `lane` of a warp holds of a matrix product's operand
// (of keys: token lane / 4, eight values from 8 (lane % 4) on; of values: tokens t, t + 1, t + 8, t + 9 with t = 2 (lane % 4) of values lane / 4 and lane / 4 + 8).
#pragma once
#include "batch_table.cuh"

#include <algorithm>

namespace {

constexpr uint32_t kPageHead = 16;                                   // bytes before a head's codes
struct PageShape { uint32_t G, dk, dv, page, shift, kp, vp, head; };      // kp, vp: padded sizes; head: bytes of a head's part; page = 1 << shift
__host__ __device__ __forceinline__ PageShape page_shape(uint32_t G, uint32_t dk, uint32_t dv, uint32_t page) {
    PageShape s;
    s.G = G; s.dk = dk; s.dv = dv; s.page = page; s.shift = page == 64 ? 6 : page == 32 ? 5 : 4;
    s.kp = (dk + 31) & ~31u; s.vp = (dv + 15) & ~15u;
    s.head = kPageHead + page * (s.kp + s.vp);
    return s;
}
__host__ __device__ __forceinline__ size_t page_bytes(const PageShape& s) { return (size_t)s.G * s.head; }
inline bool page_shape_ok(size_t G, size_t dk, size_t dv, size_t page) { return G && G <= 1024 && dk && dv && dk <= 256 && dv <= 256 && (page == 16 || page == 32 || page == 64); }
// byte of (token, dim) in a head's part
__device__ __forceinline__ uint32_t key_byte(const PageShape& s, uint32_t t, uint32_t d) { return kPageHead + ((t >> 3) * (s.kp >> 5) + (d >> 5)) * 256 + (t & 7) * 32 + (d & 31); }
__device__ __forceinline__ uint32_t value_byte(const PageShape& s, uint32_t t, uint32_t d) {
    return kPageHead + s.page * s.kp + ((t >> 4) * (s.vp >> 4) + (d >> 4)) * 256 + (4 * (d & 7) + ((t & 7) >> 1)) * 8 + 4 * ((d >> 3) & 1) + 2 * ((t >> 3) & 1) + (t & 1);
}
// The page tables [slots, most] and the pool they name pages of; ids are checked before they become addresses.
struct PagePool { const uint8_t* pages; const int32_t* table; uint32_t count, slots, most; };
__device__ __forceinline__ int32_t page_id(const PagePool& p, uint32_t slot, uint32_t nth) {
    const int32_t id = p.table[(size_t)slot * p.most + nth];
    return (uint32_t)id < p.count ? id : -1;
}
inline PagePool page_pool(const float* pages, size_t page_elems, const float* table, size_t table_elems, uint32_t most, const PageShape& s) {
    PagePool p;
    p.pages = reinterpret_cast<const uint8_t*>(pages); p.table = reinterpret_cast<const int32_t*>(table); p.most = most;
    p.count = (uint32_t)std::min<size_t>(page_elems / (page_bytes(s) / 4), 0x7fffffffu);
    p.slots = (uint32_t)std::min<size_t>(table_elems / most, 0x7fffffffu);
    return p;
}
// whether a row's words lie inside the tables (its pages are checked where they are used)
__device__ __forceinline__ bool page_row_ok(const PagePool& p, const PageShape& s, const BatchRow& w) { return (uint32_t)w.slot < p.slots && w.length >= 0 && (uint64_t)w.length <= ((uint64_t)p.most << s.shift); }

}  // namespace
inline size_t zg_page_words(size_t G, size_t dk, size_t dv, size_t page) { return page_bytes(page_shape((uint32_t)G, (uint32_t)dk, (uint32_t)dv, (uint32_t)page)) / 4; }

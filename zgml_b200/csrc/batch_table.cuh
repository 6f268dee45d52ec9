// The table of a batch (BATCH_APPEND, SHARED_ATTENTION, ADAPTER_LINEAR; layout in include/zgml_cuda.h) as the kernels read it.  It is device data that
// the host rewrites between executions of a captured program, so every word is checked here before it becomes an address.
#pragma once
#include "seq_common.cuh"

namespace {

struct BatchHead { uint32_t rows; int32_t prefix, prefix_slot; };
__device__ __forceinline__ BatchHead batch_head(const float* table, uint32_t B) {
    const int4 w = *reinterpret_cast<const int4*>(table);
    BatchHead h;
    h.rows = w.x < 0 ? 0u : min((uint32_t)w.x, B);
    h.prefix = w.y; h.prefix_slot = w.z;
    return h;
}
struct BatchRow { int32_t slot, length, adapter; };
__device__ __forceinline__ BatchRow batch_row(const float* table, uint32_t r) {
    const int4 w = *reinterpret_cast<const int4*>(table + ZG_BATCH_ROWS + (size_t)4 * r);
    BatchRow b;
    b.slot = w.x; b.length = w.y; b.adapter = w.z;
    return b;
}
// what a row with a word out of range gets: the mistake shows, and nothing out of bounds is touched
constexpr float kBatchNaN = __builtin_nanf("");

}  // namespace

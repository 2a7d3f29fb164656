// The 4-bit paged key/value cache: where a row's bytes lie (the layout is
// stated in include/freeml_cuda.h) and how a batch entry finds its rows.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fml_common.cuh"

namespace fml {

// One layer's cache as the kernels see it.
struct Kv4View
{
    const int32_t* table;      // [slots][max_pages]
    const uint32_t* lens;      // [slots]
    const uint32_t* slot_ids;  // [batch], or null: entry b is slot b
    uint32_t pages, slots, max_pages;
    uint32_t page_shift;       // page_size = 1 << page_shift
    uint32_t kv_heads;
};

// Byte offsets inside a block of page_size rows of one head.
template <int HD>
struct Kv4Block
{
    static constexpr uint32_t ROW = HD / 2;    // codes of a row
    static constexpr uint32_t META = HD / 8;   // (scale, minimum) pairs of a row
    static constexpr int NG = HD / 32;         // groups of a row
    __host__ __device__ static constexpr uint32_t bytes(uint32_t page_size) { return page_size * (HD * 5 / 4); }
    __host__ __device__ static constexpr uint32_t kmeta(uint32_t page_size) { return page_size * ROW; }
    __host__ __device__ static constexpr uint32_t v(uint32_t page_size) { return page_size * (ROW + META); }
    __host__ __device__ static constexpr uint32_t vmeta(uint32_t page_size) { return page_size * (2 * ROW + META); }
};

// Slot of batch entry b, or ~0 where it names none.
__device__ __forceinline__ uint32_t kv4_slot(const Kv4View& c, uint32_t b)
{
    const uint32_t s = c.slot_ids ? c.slot_ids[b] : b;
    return s < c.slots ? s : ~0u;
}

// Rows of a slot, never more than its table row can hold.
__device__ __forceinline__ uint32_t kv4_len(const Kv4View& c, uint32_t slot)
{
    if (slot == ~0u) return 0;
    const uint32_t n = c.lens[slot], most = c.max_pages << c.page_shift;
    return n < most ? n : most;
}

// log2 of a supported page size, or 0
inline uint32_t kv4_page_shift(uint32_t page_size)
{
    return page_size == 16 ? 4u : page_size == 32 ? 5u : page_size == 64 ? 6u : page_size == 128 ? 7u : 0u;
}

// ---- element types ----------------------------------------------------------

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

inline size_t type_bytes(int type) { return type == FML_TYPE_FP32 ? 4 : 2; }

}  // namespace fml

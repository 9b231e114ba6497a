// air_hip_kv8.hpp -- device view of the paged 8-bit KV cache (internal).
//
// A page holds [layer][KV head][block] records; a record is 16 consecutive
// tokens (a block) of one layer and KV head:
//
//   0     f32 scale of K, f32 scale of V, 56 unused bytes
//   64    f32 accumulated attention weight of each token
//   128   K codes [token / 4][dim / 16][token % 4][dim % 16]
//   ...   V codes [dim][token]
//
// The orders are those in which a wavefront feeds the matrix cores
// (attention_kv8.hip): of K, the 16 bytes of a token's 16 dims are one lane's
// A operand, and the four tokens x four dim groups that a load instruction
// takes from one block are 256 contiguous bytes; of V, a lane's operand is
// one dim of all 16 tokens, 16 contiguous bytes.  Both are loaded straight
// into registers.  Scales, weights and codes of a block share a record so
// that a token's page is found once; the scales lie in the header's first 64
// bytes, which a plain attention reads alone.
#pragma once

#include "air_hip_kernels.hpp"

#include <hip/hip_runtime.h>
#include <cstdint>

namespace air_hip {

constexpr unsigned kKv8Weights = 64;    // byte offset of the weights
constexpr unsigned kKv8Codes = 128;     // byte offset of the K codes

// A record in global memory, and loads and stores that say so: through a
// pointer that came out of memory they would be flat, which wait together
// with LDS.
typedef __attribute__((address_space(1))) unsigned char Kv8Byte;
template <typename T>
__device__ __forceinline__ T kv8_load(const Kv8Byte* p) {
    return *(const __attribute__((address_space(1))) T*)p;
}
template <typename T>
__device__ __forceinline__ void kv8_store(Kv8Byte* p, T x) {
    *(__attribute__((address_space(1))) T*)p = x;
}

// x of this lane and those below it, summed: within rows of 16 lanes, then the
// last lane of a row to the next, and of the lower half to the upper.
__device__ __forceinline__ std::uint32_t wave_sums(std::uint32_t x) {
    x += __builtin_amdgcn_update_dpp(0u, x, 0x111, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x112, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x118, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x142, 0xa, 0xf, false);
    return x + __builtin_amdgcn_update_dpp(0u, x, 0x143, 0xc, 0xf, false);
}

// Entry of a page table that names block `block`'s page.
__device__ __forceinline__ std::uint32_t kv8_slot(const Kv8Geometry& g, std::uint32_t block) {
    return g.page_magic == 0u ? block : __umulhi(block, g.page_magic);
}

// Record of block `block` in the page that entry `slot` of its table names;
// null when the pool holds no such page.
__device__ __forceinline__ Kv8Byte* kv8_record_in(const Kv8Geometry& g, std::int32_t page, std::uint32_t slot,
                                                  std::uint32_t layer, std::uint32_t head, std::uint32_t block) {
    if (page < 0 || static_cast<std::uint32_t>(page) >= g.pool_pages) return nullptr;
    std::uint32_t p = static_cast<std::uint32_t>(page);
    unsigned char* base = g.pool;
    if (g.chunks != nullptr) {
        base = g.chunks[p >> g.chunk_shift];
        if (base == nullptr) return nullptr;
        p &= (1u << g.chunk_shift) - 1u;
    }
    const std::uint32_t offset = (layer * g.kv_heads + head) * g.head_bytes + (block - slot * g.page_blocks) * g.record_bytes;
    return (Kv8Byte*)(base + static_cast<std::uint64_t>(p) * g.page_bytes + offset);
}

// Record of block `block` of the sequence with this page table, or null when
// the table does not name a page of the pool.
__device__ __forceinline__ Kv8Byte* kv8_record(const Kv8Geometry& g, const std::int32_t* table, std::uint32_t layer,
                                               std::uint32_t head, std::uint32_t block) {
    const std::uint32_t slot = kv8_slot(g, block);
    if (slot >= g.max_pages) return nullptr;
    return kv8_record_in(g, table[slot], slot, layer, head, block);
}

// Offset of (token, dim) in a record's K and V codes.
__device__ __forceinline__ unsigned kv8_k_offset(unsigned head_dim, unsigned token, unsigned dim) {
    return kKv8Codes + ((token >> 2) * (head_dim >> 4) + (dim >> 4)) * 64u + (token & 3u) * 16u + (dim & 15u);
}
__device__ __forceinline__ unsigned kv8_v_offset(unsigned head_dim, unsigned token, unsigned dim) {
    return kKv8Codes + kKv8Block * head_dim + dim * kKv8Block + token;
}

// The code nearest to q (ties to even, clamped) as a byte, and what four
// codes of a dword stand for.  i8 codes are held with an excess of 128, which
// makes the f16 matrix operand one byte permute and one packed subtract.
template <int TYPE>
__device__ __forceinline__ std::uint32_t kv8_encode(float q) {
    if constexpr (TYPE == kKv8I8) {
        const float c = fminf(fmaxf(rintf(q), -127.0f), 127.0f);
        return static_cast<std::uint32_t>(static_cast<int>(c) + 128);
    } else {
        const float c = fminf(fmaxf(q, -448.0f), 448.0f);
        return static_cast<std::uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, c, 0, false)) & 0xffu;
    }
}
template <int TYPE>
__device__ __forceinline__ float kv8_value(std::uint32_t code) {
    if constexpr (TYPE == kKv8I8) {
        return static_cast<float>(static_cast<int>(code & 0xffu) - 128);
    } else {
        return __builtin_amdgcn_cvt_f32_fp8(code, 0);
    }
}
template <int TYPE>
constexpr std::uint32_t kv8_zero_code() {
    return TYPE == kKv8I8 ? 128u : 0u;
}

} // namespace air_hip

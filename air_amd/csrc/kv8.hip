// kv8.hip -- the paged 8-bit KV cache: quantising append, read, eviction.
//
// A block (16 tokens of one layer and KV head) holds its K and its V codes
// under one f32 scale each; a value is code * scale.  The scale of values
// with largest magnitude A is A times the f32 nearest to 1 / qmax (127 for i8,
// 448 for e4m3), a code the nearest to x / scale (f32 quotient, ties to even).  A block that
// takes a non-finite value gets a NaN scale and reads as NaN until it is
// begun anew, so a broken model shows in its logits as it does over the f32
// pool instead of turning into large finite keys.
#include "air_hip_device.hpp"
#include "air_hip_kernels.hpp"
#include "air_hip_kv8.hpp"

namespace air_hip {
namespace {

__device__ __forceinline__ constexpr float kv8_unit(int type) { return type == kKv8I8 ? 1.0f / 127.0f : 1.0f / 448.0f; }

// Code of x in a block of scale s: zero where the scale holds nothing (zero:
// all values are zero; NaN: the block is poisoned).
template <int TYPE>
__device__ __forceinline__ std::uint32_t kv8_code(float x, float s) {
    return s > 0.0f ? kv8_encode<TYPE>(x / s) : kv8_zero_code<TYPE>();
}

// A held code under a scale that grew by 1 / ratio.
template <int TYPE>
__device__ __forceinline__ std::uint32_t kv8_recode(std::uint32_t code, float ratio) {
    return kv8_encode<TYPE>(kv8_value<TYPE>(code) * ratio);
}

__device__ __forceinline__ std::uint32_t wave_max_u32(std::uint32_t v) {
    for (int off = 32; off > 0; off >>= 1) {
        const std::uint32_t o = static_cast<std::uint32_t>(__shfl_xor(static_cast<int>(v), off));
        v = o > v ? o : v;
    }
    return v;
}

__device__ __forceinline__ float nan_f32() { return __builtin_nanf(""); }

// One workgroup per (row, KV head); the row whose block no earlier row of the
// call names stores every row of that block (the last row of a slot wins), so
// rows may come in any order and a block has one writer.  Threads [0, D) own
// K: (token, 16 dims), one 16-byte store each; threads [D, 2 D) own V: one
// dim of all 16 tokens.  The magnitudes meet as the bit patterns of |x|,
// whose unsigned order puts infinities and NaN above every finite value.
template <int TYPE, unsigned D>
__global__ __launch_bounds__(2 * D) void kv8_append_kernel(Kv8Geometry g, const float* __restrict__ qkv,
                                                           std::uint64_t stride, std::uint64_t q_width,
                                                           std::uint32_t m, const std::int32_t* __restrict__ positions,
                                                           const std::int32_t* __restrict__ tables,
                                                           std::uint32_t layer) {
#pragma clang fp contract(off)
    __shared__ int winner[kKv8Block];
    __shared__ int earlier;
    __shared__ std::uint32_t wave_top[2 * D / 64];
    const std::uint32_t r = blockIdx.x, head = blockIdx.y;
    const unsigned tid = threadIdx.x;
    const auto record_of = [&](std::uint32_t row, std::int32_t pos) __attribute__((always_inline)) {
        return pos < 0 ? nullptr
                       : kv8_record(g, tables + static_cast<std::uint64_t>(row) * g.max_pages, layer, head,
                                    static_cast<std::uint32_t>(pos) / kKv8Block);
    };
    unsigned char* const rec = record_of(r, positions[r]);
    if (rec == nullptr) return;
    // In a prompt the row before names the same block for 15 of 16 rows.
    if (r > 0u && record_of(r - 1u, positions[r - 1u]) == rec) return;
    if (tid < kKv8Block) winner[tid] = -1;
    if (tid == 0u) earlier = 0;
    __syncthreads();
    for (std::uint32_t o = tid; o < m; o += 2u * D) {
        const std::int32_t pos = positions[o];
        if (record_of(o, pos) != rec) continue;
        if (o < r) {
            earlier = 1;
        } else {
            atomicMax(&winner[static_cast<std::uint32_t>(pos) % kKv8Block], static_cast<int>(o));
        }
    }
    __syncthreads();
    if (earlier != 0) return;
    unsigned first = 0u;
    while (winner[first] < 0) ++first;   // row r itself is in

    const bool value = tid >= D;
    const unsigned part = value ? tid - D : tid;
    const unsigned token = part / (D / 16u), chunk = part % (D / 16u);   // of a K thread
    float x[16];
    std::uint32_t top = 0u;
    const float* const base = qkv + q_width + (value ? static_cast<std::uint64_t>(g.kv_heads) * D : 0u) +
                              static_cast<std::uint64_t>(head) * D;
#pragma unroll
    for (unsigned i = 0; i < 16u; ++i) {
        const int row = winner[value ? i : token];
        x[i] = row >= 0 ? base[static_cast<std::uint64_t>(row) * stride + (value ? part : chunk * 16u + i)] : 0.0f;
        const std::uint32_t mag = __float_as_uint(x[i]) & 0x7fffffffu;
        top = mag > top ? mag : top;
    }
    float* const scale_at = reinterpret_cast<float*>(rec) + (value ? 1 : 0);
    const float old_scale = *scale_at;
    top = wave_max_u32(top);
    if ((tid & 63u) == 0u) wave_top[tid >> 6] = top;
    __syncthreads();   // also: every thread has the old scale before it is replaced
    top = 0u;
#pragma unroll
    for (unsigned w = 0; w < D / 64u; ++w) {
        const std::uint32_t t = wave_top[(value ? D / 64u : 0u) + w];
        top = t > top ? t : top;
    }
    const float need = top >= 0x7f800000u ? nan_f32() : __uint_as_float(top) * kv8_unit(TYPE);
    const bool held = first > 0u;
    // !(need <= old): a NaN need replaces the scale, a NaN scale stays.
    const bool grows = held && old_scale == old_scale && !(need <= old_scale);
    const float scale = held && !grows ? old_scale : need;
    const float ratio = grows && scale > 0.0f ? old_scale / scale : 1.0f;
    const unsigned at = value ? kv8_v_offset(D, 0u, part) : kv8_k_offset(D, token, chunk * 16u);
    u32x4* const codes_at = reinterpret_cast<u32x4*>(rec + at);
    u32x4 codes = *codes_at;
#pragma unroll
    for (unsigned i = 0; i < 16u; ++i) {
        const unsigned t = value ? i : token;
        const unsigned shift = 8u * (i & 3u);
        const std::uint32_t was = (codes[i >> 2] >> shift) & 0xffu;
        std::uint32_t now = was;
        if (winner[t] >= 0) {
            now = kv8_code<TYPE>(x[i], scale);
        } else if (t < first && grows) {
            now = kv8_recode<TYPE>(was, ratio);
        }
        codes[i >> 2] = (codes[i >> 2] & ~(0xffu << shift)) | (now << shift);
    }
    *codes_at = codes;
    if (part == 0u) *scale_at = scale;
    if (tid < kKv8Block && winner[tid] >= 0) {
        reinterpret_cast<float*>(rec + kKv8Weights)[tid] = 0.0f;   // a new token has gathered no weight
    }
}

// Tokens starts[i] .. starts[i] + lengths[i] - 1 of every sequence as f32
// rows; one workgroup per (block, KV head, sequence and layer), a thread per
// four dims of a token.
template <int TYPE>
__global__ __launch_bounds__(256) void kv8_read_kernel(Kv8Geometry g, std::uint32_t seqs,
                                                       const std::int32_t* __restrict__ starts,
                                                       const std::int32_t* __restrict__ lengths,
                                                       const std::int32_t* __restrict__ tables, std::uint32_t layer,
                                                       std::uint64_t max_tokens, float* __restrict__ k,
                                                       float* __restrict__ v, float* __restrict__ weights) {
    const std::uint32_t head = blockIdx.y;
    const std::uint32_t seq = blockIdx.z % seqs, l = blockIdx.z / seqs;
    const std::int64_t start = starts ? starts[seq] : 0;
    std::int64_t count = lengths[seq];
    if (start < 0 || count <= 0) return;
    if (count > static_cast<std::int64_t>(max_tokens)) count = static_cast<std::int64_t>(max_tokens);
    const std::int64_t block = start / kKv8Block + blockIdx.x;
    const std::int64_t base = block * kKv8Block;   // first token of the block
    if (base >= start + count || block > 0x7fffffff / static_cast<std::int64_t>(kKv8Block)) return;
    const unsigned char* const rec = kv8_record(g, tables + static_cast<std::uint64_t>(seq) * g.max_pages, layer + l,
                                                head, static_cast<std::uint32_t>(block));
    if (rec == nullptr) return;
    const unsigned d = g.head_dim, quads = d / 4u;
    const std::uint64_t row0 = (static_cast<std::uint64_t>(l) * seqs + seq) * max_tokens;
    const std::uint64_t width = static_cast<std::uint64_t>(g.kv_heads) * d;
    const float ks = reinterpret_cast<const float*>(rec)[0], vs = reinterpret_cast<const float*>(rec)[1];
    for (unsigned idx = threadIdx.x; idx < kKv8Block * quads; idx += 256u) {
        const unsigned token = idx / quads, dim = idx % quads * 4u;
        const std::int64_t t = base + token;
        if (t < start || t >= start + count) continue;
        const std::uint64_t at = (row0 + static_cast<std::uint64_t>(t - start)) * width +
                                 static_cast<std::uint64_t>(head) * d + dim;
        if (k) {
            const std::uint32_t c = *reinterpret_cast<const std::uint32_t*>(rec + kv8_k_offset(d, token, dim));
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i) k[at + i] = kv8_value<TYPE>(c >> (8u * i)) * ks;
        }
        if (v) {
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i) v[at + i] = kv8_value<TYPE>(rec[kv8_v_offset(d, token, dim + i)]) * vs;
        }
    }
    if (weights && threadIdx.x < kKv8Block) {
        const std::int64_t t = base + threadIdx.x;
        if (t >= start && t < start + count) {
            weights[(row0 + static_cast<std::uint64_t>(t - start)) * g.kv_heads + head] =
                reinterpret_cast<const float*>(rec + kKv8Weights)[threadIdx.x];
        }
    }
}

// ---- eviction ----------------------------------------------------------------

constexpr unsigned kSelectThreads = 256;

// Weights as unsigned integers of the same order; NaN (and a token whose page
// is absent) lowest, the two zeros equal.
__device__ __forceinline__ std::uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const std::uint32_t b = __float_as_uint(w + 0.0f);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ std::int64_t held_tokens(const Kv8Geometry& g, std::int32_t length, std::uint64_t max_tokens) {
    std::uint64_t n = length < 0 ? 0u : static_cast<std::uint64_t>(length);
    if (n > max_tokens) n = max_tokens;
    const std::uint64_t most = static_cast<std::uint64_t>(g.max_pages) * g.page_blocks * kKv8Block;
    return static_cast<std::int64_t>(n < most ? n : most);
}

// The tokens a (sequence, layer, KV head) keeps, ascending, -1 behind them.
// The want-th largest key of the middle tokens is found byte by byte from the
// top (a histogram of the next byte over the keys that agree so far); then one
// pass in token order writes the first keep_first, every larger key, as many
// equal ones as are still wanted (the lowest tokens) and the last keep_last.
__global__ __launch_bounds__(kSelectThreads) void kv8_select_kernel(
    Kv8Geometry g, const std::int32_t* __restrict__ lengths, const std::int32_t* __restrict__ tables,
    std::uint32_t layer, std::uint32_t layers, std::uint32_t keep_first, std::uint32_t keep_last, std::uint32_t budget,
    std::uint64_t max_tokens, std::int32_t* __restrict__ kept) {
    constexpr unsigned kWaves = kSelectThreads / 64u;
    __shared__ std::uint32_t bins[256];
    __shared__ std::uint32_t found_prefix, found_want;
    __shared__ std::uint32_t wave_above[kWaves], wave_equal[kWaves];
    const std::uint32_t head = blockIdx.x, l = blockIdx.y, seq = blockIdx.z;
    const unsigned tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const std::int32_t* const table = tables + static_cast<std::uint64_t>(seq) * g.max_pages;
    std::int32_t* const out = kept + ((static_cast<std::uint64_t>(seq) * layers + l) * g.kv_heads + head) * budget;
    const std::int64_t n = held_tokens(g, lengths[seq], max_tokens);
    if (n <= static_cast<std::int64_t>(budget)) {
        for (std::int64_t i = tid; i < static_cast<std::int64_t>(budget); i += kSelectThreads) {
            out[i] = i < n ? static_cast<std::int32_t>(i) : -1;
        }
        return;
    }
    const auto key_of = [&](std::int64_t t) __attribute__((always_inline)) -> std::uint32_t {
        const unsigned char* const rec =
            kv8_record(g, table, layer + l, head, static_cast<std::uint32_t>(t / kKv8Block));
        return rec ? weight_key(reinterpret_cast<const float*>(rec + kKv8Weights)[t % kKv8Block]) : 0u;
    };
    const std::int64_t lo = keep_first, hi = n - keep_last;
    const std::uint32_t want = budget - keep_first - keep_last;   // of the hi - lo > want middle tokens
    std::uint32_t prefix = 0u, left = want;
    if (want > 0u) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (unsigned b = tid; b < 256u; b += kSelectThreads) bins[b] = 0u;
            __syncthreads();
            for (std::int64_t t = lo + tid; t < hi; t += kSelectThreads) {
                const std::uint32_t key = key_of(t);
                // Shifts of 32 are undefined: the first round takes every key.
                if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&bins[(key >> shift) & 255u], 1u);
            }
            __syncthreads();
            if (tid == 0u) {
                std::uint32_t rest = left;
                int b = 255;
                while (b > 0 && bins[b] < rest) rest -= bins[b--];
                found_prefix = prefix | static_cast<std::uint32_t>(b) << shift;
                found_want = rest;
            }
            __syncthreads();
            prefix = found_prefix;
            left = found_want;
        }
    }
    // prefix is the want-th largest key, left how many keys equal to it stay.
    for (std::int64_t i = tid; i < keep_first; i += kSelectThreads) out[i] = static_cast<std::int32_t>(i);
    for (std::int64_t i = tid; i < keep_last; i += kSelectThreads) {
        out[budget - keep_last + i] = static_cast<std::int32_t>(hi + i);
    }
    std::uint32_t base_above = 0u, base_equal = 0u;   // larger and equal keys before this round
    for (std::int64_t t0 = lo; want > 0u && t0 < hi; t0 += kSelectThreads) {
        const std::int64_t t = t0 + tid;
        const std::uint32_t key = t < hi ? key_of(t) : 0u;
        const bool above = t < hi && key > prefix, equal = t < hi && key == prefix;
        const std::uint64_t above_mask = __ballot(above), equal_mask = __ballot(equal);
        if (lane == 0u) {
            wave_above[wave] = static_cast<std::uint32_t>(__popcll(above_mask));
            wave_equal[wave] = static_cast<std::uint32_t>(__popcll(equal_mask));
        }
        __syncthreads();
        std::uint32_t a = base_above, e = base_equal, all_above = 0u, all_equal = 0u;
        for (unsigned w = 0; w < kWaves; ++w) {
            if (w < wave) {
                a += wave_above[w];
                e += wave_equal[w];
            }
            all_above += wave_above[w];
            all_equal += wave_equal[w];
        }
        const std::uint64_t below = (1ull << lane) - 1u;
        a += static_cast<std::uint32_t>(__popcll(above_mask & below));
        e += static_cast<std::uint32_t>(__popcll(equal_mask & below));
        if (above || (equal && e < left)) {
            out[keep_first + a + (e < left ? e : left)] = static_cast<std::int32_t>(t);
        }
        base_above += all_above;
        base_equal += all_equal;
        __syncthreads();
    }
}

// Gathers the kept tokens of a (sequence, layer, KV head) into blocks of the
// new table.  A block's scale is the largest of its tokens' scales, so a
// block whose tokens come from one block keeps its codes, and others are
// rounded once.  Threads as in the append.  Where the new table is the old
// one (in place) a workgroup takes all blocks in ascending order: block b's
// tokens come from blocks >= b, so what it overwrites no later block reads,
// and it reads its 16 tokens before it writes.
template <int TYPE, unsigned D>
__global__ __launch_bounds__(2 * D) void kv8_compact_kernel(Kv8Geometry g, const std::int32_t* lengths,
                                                            const std::int32_t* tables, const std::int32_t* new_tables,
                                                            std::uint32_t layer, std::uint32_t layers,
                                                            std::uint32_t heads, std::uint32_t budget,
                                                            std::uint64_t max_tokens, const std::int32_t* kept,
                                                            bool in_place) {
#pragma clang fp contract(off)
    __shared__ const unsigned char* source[kKv8Block];
    __shared__ std::uint32_t source_slot[kKv8Block];
    __shared__ float source_scale[2][kKv8Block];
    __shared__ float source_weight[kKv8Block];
    const std::uint32_t head = blockIdx.y % heads, l = blockIdx.y / heads, seq = blockIdx.z;
    const std::int64_t n = held_tokens(g, lengths[seq], max_tokens);
    if (in_place && n <= static_cast<std::int64_t>(budget)) return;   // everything stays where it is
    const unsigned tid = threadIdx.x;
    const bool value = tid >= D;
    const unsigned part = value ? tid - D : tid;
    const unsigned token = part / (D / 16u), chunk = part % (D / 16u);
    const std::int32_t* const table = tables + static_cast<std::uint64_t>(seq) * g.max_pages;
    const std::int32_t* const new_table = new_tables + static_cast<std::uint64_t>(seq) * g.max_pages;
    const std::int32_t* const list =
        kept + ((static_cast<std::uint64_t>(seq) * layers + l) * g.kv_heads + head) * budget;
    const std::uint32_t tokens = n < static_cast<std::int64_t>(budget) ? static_cast<std::uint32_t>(n) : budget;
    const std::uint32_t blocks = (tokens + kKv8Block - 1u) / kKv8Block;
    for (std::uint32_t b = blockIdx.x; b < blocks; b += gridDim.x) {
        if (tid < kKv8Block) {
            const std::uint32_t i = b * kKv8Block + tid;
            const std::int32_t t = i < tokens ? list[i] : -1;
            const unsigned char* src = nullptr;
            float s0 = 0.0f, s1 = 0.0f, w = 0.0f;
            unsigned slot = 0u;
            if (t >= 0) {
                slot = static_cast<std::uint32_t>(t) % kKv8Block;
                src = kv8_record(g, table, layer + l, head, static_cast<std::uint32_t>(t) / kKv8Block);
                if (src) {
                    s0 = reinterpret_cast<const float*>(src)[0];
                    s1 = reinterpret_cast<const float*>(src)[1];
                    w = reinterpret_cast<const float*>(src + kKv8Weights)[slot];
                }
            }
            source[tid] = src;
            source_slot[tid] = slot;
            source_scale[0][tid] = s0;
            source_scale[1][tid] = s1;
            source_weight[tid] = w;
        }
        __syncthreads();
        const float* const scales = source_scale[value ? 1 : 0];
        float scale = 0.0f;
#pragma unroll
        for (unsigned i = 0; i < kKv8Block; ++i) {
            // Once NaN it stays: a poisoned token poisons its new block.
            if (scale == scale && !(scales[i] <= scale)) scale = scales[i];
        }
        u32x4 codes;
#pragma unroll
        for (unsigned i = 0; i < 4u; ++i) codes[i] = kv8_zero_code<TYPE>() * 0x01010101u;
        if (value) {
#pragma unroll
            for (unsigned i = 0; i < 16u; ++i) {
                if (source[i] == nullptr) continue;
                const std::uint32_t was = source[i][kv8_v_offset(D, source_slot[i], part)];
                const std::uint32_t now =
                    scales[i] == scale ? was : kv8_recode<TYPE>(was, scale > 0.0f ? scales[i] / scale : 0.0f);
                codes[i >> 2] = (codes[i >> 2] & ~(0xffu << (8u * (i & 3u)))) | now << (8u * (i & 3u));
            }
        } else if (source[token] != nullptr) {
            codes = *reinterpret_cast<const u32x4*>(source[token] + kv8_k_offset(D, source_slot[token], chunk * 16u));
            if (scales[token] != scale) {
                const float ratio = scale > 0.0f ? scales[token] / scale : 0.0f;
#pragma unroll
                for (unsigned i = 0; i < 16u; ++i) {
                    const std::uint32_t was = (codes[i >> 2] >> (8u * (i & 3u))) & 0xffu;
                    codes[i >> 2] = (codes[i >> 2] & ~(0xffu << (8u * (i & 3u)))) |
                                    kv8_recode<TYPE>(was, ratio) << (8u * (i & 3u));
                }
            }
        }
        __syncthreads();   // the block's tokens are read: in place, what they share with it may go
        unsigned char* const dst = kv8_record(g, new_table, layer + l, head, b);
        if (dst != nullptr) {
            const unsigned at = value ? kv8_v_offset(D, 0u, part) : kv8_k_offset(D, token, chunk * 16u);
            *reinterpret_cast<u32x4*>(dst + at) = codes;
            if (part == 0u) reinterpret_cast<float*>(dst)[value ? 1 : 0] = scale;
            if (tid < kKv8Block) reinterpret_cast<float*>(dst + kKv8Weights)[tid] = source_weight[tid];
        }
        __syncthreads();   // the lists are read before the next block replaces them
    }
}

} // namespace

hipError_t launch_kv8_append(const Kv8Geometry& g, const float* qkv, std::uint64_t stride, std::uint64_t q_width,
                             std::uint32_t m, const std::int32_t* positions, const std::int32_t* tables,
                             std::uint32_t layer, hipStream_t stream) {
    const dim3 grid(m, g.kv_heads);
#define AIR_KV8_APPEND(T, D)                                                                                     \
    hipLaunchKernelGGL((kv8_append_kernel<T, D>), grid, dim3(2 * D), 0, stream, g, qkv, stride, q_width, m, positions, \
                       tables, layer)
    if (g.type == kKv8I8) {
        if (g.head_dim == 128u) AIR_KV8_APPEND(kKv8I8, 128);
        else AIR_KV8_APPEND(kKv8I8, 64);
    } else {
        if (g.head_dim == 128u) AIR_KV8_APPEND(kKv8E4M3, 128);
        else AIR_KV8_APPEND(kKv8E4M3, 64);
    }
#undef AIR_KV8_APPEND
    return hipGetLastError();
}

hipError_t launch_kv8_read(const Kv8Geometry& g, std::uint32_t seqs, const std::int32_t* starts,
                           const std::int32_t* lengths, const std::int32_t* tables, std::uint32_t layer,
                           std::uint32_t layers, std::uint64_t max_tokens, float* k, float* v, float* weights,
                           hipStream_t stream) {
    // A start inside a block makes the tokens span one more.
    const std::uint64_t blocks = (max_tokens + kKv8Block - 1u) / kKv8Block + (starts ? 1u : 0u);
    const dim3 grid(static_cast<unsigned>(blocks), g.kv_heads, seqs * layers);
    if (g.type == kKv8I8) {
        hipLaunchKernelGGL(kv8_read_kernel<kKv8I8>, grid, dim3(256), 0, stream, g, seqs, starts, lengths, tables, layer,
                           max_tokens, k, v, weights);
    } else {
        hipLaunchKernelGGL(kv8_read_kernel<kKv8E4M3>, grid, dim3(256), 0, stream, g, seqs, starts, lengths, tables,
                           layer, max_tokens, k, v, weights);
    }
    return hipGetLastError();
}

hipError_t launch_kv8_evict(const Kv8Geometry& g, std::uint32_t seqs, const std::int32_t* lengths,
                            const std::int32_t* tables, const std::int32_t* new_tables, std::uint32_t layer,
                            std::uint32_t layers, std::uint32_t keep_first, std::uint32_t keep_last,
                            std::uint32_t budget, std::uint64_t max_tokens, std::int32_t* kept, hipStream_t stream) {
    hipLaunchKernelGGL(kv8_select_kernel, dim3(g.kv_heads, layers, seqs), dim3(kSelectThreads), 0, stream, g, lengths,
                       tables, layer, layers, keep_first, keep_last, budget, max_tokens, kept);
    const bool in_place = tables == new_tables;
    const std::uint64_t most = budget < max_tokens ? budget : max_tokens;
    const std::uint32_t blocks = static_cast<std::uint32_t>((most + kKv8Block - 1u) / kKv8Block);
    const dim3 grid(in_place ? 1u : blocks, g.kv_heads * layers, seqs);
#define AIR_KV8_COMPACT(T, D)                                                                                      \
    hipLaunchKernelGGL((kv8_compact_kernel<T, D>), grid, dim3(2 * D), 0, stream, g, lengths, tables, new_tables, layer, \
                       layers, g.kv_heads, budget, max_tokens, kept, in_place)
    if (g.type == kKv8I8) {
        if (g.head_dim == 128u) AIR_KV8_COMPACT(kKv8I8, 128);
        else AIR_KV8_COMPACT(kKv8I8, 64);
    } else {
        if (g.head_dim == 128u) AIR_KV8_COMPACT(kKv8E4M3, 128);
        else AIR_KV8_COMPACT(kKv8E4M3, 64);
    }
#undef AIR_KV8_COMPACT
    return hipGetLastError();
}

} // namespace air_hip

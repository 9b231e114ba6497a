// kv8.hip -- the paged 8-bit KV cache: quantising append, read, eviction.
//
// A block (16 tokens of one layer and KV head) holds its K and its V codes
// under one f32 scale each; a value is code * scale.  The scale of values
// with largest magnitude A is A times the f32 nearest to 1 / qmax (127 for i8,
// 448 for e4m3), a code the nearest to x / scale (f32 quotient, ties to even).
// A block that takes a non-finite value gets a NaN scale and reads as NaN until
// it is begun anew, so a broken model shows in its logits as it does over the
// f32 pool instead of turning into large finite keys.
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
// Latency bounds it (a decode step stores 2 KB a row, a prompt's 264 blocks
// take 8 dependent loads): the block's codes and scale and the rows that a
// decode step or a prompt stores in it (the next rows in the next slots) are
// asked for before the other rows are looked through.  32 rows of 4 KV heads
// of 128 dims take 7.4 us, two prompts of 509 rows 13.8 (1.4 and 4.4 more with
// the loads one after the other): 3.5 the launch with the 15 of 16 rows that
// only find that their block has its writer (several rows a workgroup, in a
// loop: 22), 1.4 the look at the other rows, the rest a writer's own waits.
template <int TYPE, unsigned D>
__global__ __launch_bounds__(2 * D) void kv8_append_kernel(Kv8Geometry g, const float* __restrict__ qkv,
                                                           std::uint64_t stride, std::uint64_t q_width,
                                                           std::uint32_t m, const std::int32_t* __restrict__ positions,
                                                           const std::int32_t* __restrict__ tables,
                                                           std::uint32_t layer, bool aligned) {
#pragma clang fp contract(off)
    constexpr unsigned kThreads = 2 * D;
    constexpr unsigned kAtOnce = 4;       // rows a thread looks through at a time
    __shared__ int winner[kKv8Block];
    __shared__ int earlier;
    __shared__ std::uint32_t wave_top[kThreads / 64];
    const std::uint32_t r = blockIdx.x, head = blockIdx.y;
    const unsigned tid = threadIdx.x;
    const bool value = tid >= D;
    const unsigned part = value ? tid - D : tid;
    const unsigned token = part / (D / 16u), chunk = part % (D / 16u);   // of a K thread
    const float* const base = qkv + q_width + (value ? static_cast<std::uint64_t>(g.kv_heads) * D : 0u) +
                              static_cast<std::uint64_t>(head) * D;
    // What this thread stores of row `row` in its token (K: 16 dims; V: one).
    const auto load_row = [&](std::uint32_t row, float* x) __attribute__((always_inline)) {
        const float* const src = base + static_cast<std::uint64_t>(row) * stride + chunk * 16u;
        if (aligned) {
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i) {
                const float4 f = reinterpret_cast<const float4*>(src)[i];
                x[4u * i] = f.x;
                x[4u * i + 1u] = f.y;
                x[4u * i + 2u] = f.z;
                x[4u * i + 3u] = f.w;
            }
        } else {
#pragma unroll
            for (unsigned i = 0; i < 16u; ++i) x[i] = src[i];
        }
    };
    const auto page_of = [&](std::uint32_t row, std::int32_t pos, std::uint32_t& slot) __attribute__((always_inline)) {
        slot = pos < 0 ? 0u : kv8_slot(g, static_cast<std::uint32_t>(pos) / kKv8Block);
        return pos < 0 || slot >= g.max_pages ? -1 : tables[static_cast<std::uint64_t>(row) * g.max_pages + slot];
    };
    // Two rows name one block if they name one page and its same block.
    const auto place_of = [&](std::int32_t pos, std::uint32_t slot) __attribute__((always_inline)) {
        return static_cast<std::uint32_t>(pos) / kKv8Block - slot * g.page_blocks;
    };
    // In a small call the other rows' pages are asked for at once.
    const bool small = m <= kThreads;
    std::int32_t first_pos = -1, first_page = -1;
    std::uint32_t first_slot = 0u;
    if (small && tid < m) {
        first_pos = positions[tid];
        first_page = page_of(tid, first_pos, first_slot);
    }
    const std::int32_t pos = positions[r], pos_before = r > 0u ? positions[r - 1u] : -1;
    std::uint32_t slot, slot_before;
    const std::int32_t page = page_of(r, pos, slot), page_before = page_of(r > 0u ? r - 1u : 0u, pos_before, slot_before);
    if (page < 0) return;
    const std::uint32_t place = place_of(pos, slot);
    // In a prompt the row before names the same block for 15 of 16 rows.
    if (page_before == page && place_of(pos_before, slot_before) == place) return;
    Kv8Byte* const rec = kv8_record_in(g, page, slot, layer, head, static_cast<std::uint32_t>(pos) / kKv8Block);
    if (rec == nullptr) return;
    const unsigned at = value ? kv8_v_offset(D, 0u, part) : kv8_k_offset(D, token, chunk * 16u);
    u32x4 codes = kv8_load<u32x4>(rec + at);
    Kv8Byte* const scale_at = rec + (value ? 4 : 0);
    const float old_scale = kv8_load<float>(scale_at);
    const unsigned own = static_cast<std::uint32_t>(pos) % kKv8Block;
    // The row that slot t takes if rows and slots go on together.
    const auto next_row = [&](unsigned t) __attribute__((always_inline)) -> int {
        return t >= own && t - own < m - r ? static_cast<int>(r + t - own) : -1;
    };
    float x[16];
    if (value) {
#pragma unroll
        for (unsigned i = 0; i < 16u; ++i) {
            const int row = next_row(i);
            x[i] = row >= 0 ? base[static_cast<std::uint64_t>(row) * stride + part] : 0.0f;
        }
    } else if (const int row = next_row(token); row >= 0) {
        load_row(static_cast<std::uint32_t>(row), x);
    } else {
#pragma unroll
        for (unsigned i = 0; i < 16u; ++i) x[i] = 0.0f;
    }
    if (tid < kKv8Block) winner[tid] = -1;
    if (tid == 0u) earlier = 0;
    __syncthreads();
    const auto look_at = [&](std::uint32_t o, std::int32_t their_pos, std::int32_t their_page, std::uint32_t their_slot)
                             __attribute__((always_inline)) {
        if (their_page != page || place_of(their_pos, their_slot) != place) return;
        if (o < r) {
            earlier = 1;
        } else {
            atomicMax(&winner[static_cast<std::uint32_t>(their_pos) % kKv8Block], static_cast<int>(o));
        }
    };
    if (small) {
        look_at(tid, first_pos, first_page, first_slot);
    } else {
        for (std::uint32_t o0 = tid; o0 < m; o0 += kAtOnce * kThreads) {
            std::int32_t their_pos[kAtOnce], their_page[kAtOnce];
            std::uint32_t their_slot[kAtOnce];
#pragma unroll
            for (unsigned j = 0; j < kAtOnce; ++j) {
                const std::uint32_t o = o0 + j * kThreads;
                their_pos[j] = o < m ? positions[o] : -1;
            }
#pragma unroll
            for (unsigned j = 0; j < kAtOnce; ++j) {
                const std::uint32_t o = o0 + j * kThreads;
                their_page[j] = page_of(o < m ? o : 0u, their_pos[j], their_slot[j]);
            }
#pragma unroll
            for (unsigned j = 0; j < kAtOnce; ++j) look_at(o0 + j * kThreads, their_pos[j], their_page[j], their_slot[j]);
        }
    }
    __syncthreads();
    if (earlier != 0) return;
    unsigned first = 0u;
    while (winner[first] < 0) ++first;   // row r itself is in
    if (value) {
#pragma unroll
        for (unsigned i = 0; i < 16u; ++i) {
            const int row = winner[i];
            if (row != next_row(i)) x[i] = row >= 0 ? base[static_cast<std::uint64_t>(row) * stride + part] : 0.0f;
        }
    } else if (const int row = winner[token]; row != next_row(token)) {
        if (row >= 0) {
            load_row(static_cast<std::uint32_t>(row), x);
        } else {
#pragma unroll
            for (unsigned i = 0; i < 16u; ++i) x[i] = 0.0f;
        }
    }
    std::uint32_t top = 0u;
#pragma unroll
    for (unsigned i = 0; i < 16u; ++i) {
        const std::uint32_t mag = __float_as_uint(x[i]) & 0x7fffffffu;
        top = mag > top ? mag : top;
    }
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
    kv8_store(rec + at, codes);
    if (part == 0u) kv8_store(scale_at, scale);
    if (tid < kKv8Block && winner[tid] >= 0) {
        kv8_store(rec + kKv8Weights + 4u * tid, 0.0f);   // a new token has gathered no weight
    }
}

// Tokens starts[i] .. starts[i] + lengths[i] - 1 of every sequence as f32
// rows; one workgroup per (block, KV head, sequence and layer).  Half of the
// threads read K, half V, each four tokens of four dims: four dwords of codes
// and four 16-byte stores, a token's stores of a wave being contiguous.  The
// f32 rows bound it: 24 sequences and layers of 1024 tokens, 4 KV heads of 128
// dims, 96 MB written in 25 us, 4.9 TB/s with the codes, a large copy's rate.
template <int TYPE, unsigned D>
__global__ __launch_bounds__(2 * D) void kv8_read_kernel(Kv8Geometry g, std::uint32_t seqs,
                                                         const std::int32_t* __restrict__ starts,
                                                         const std::int32_t* __restrict__ lengths,
                                                         const std::int32_t* __restrict__ tables, std::uint32_t layer,
                                                         std::uint64_t max_tokens, float* __restrict__ k,
                                                         float* __restrict__ v, float* __restrict__ weights,
                                                         bool aligned) {
    const std::uint32_t head = blockIdx.y;
    const std::uint32_t seq = blockIdx.z % seqs, l = blockIdx.z / seqs;
    const std::int64_t start = starts ? starts[seq] : 0;
    std::int64_t count = lengths[seq];
    if (start < 0 || count <= 0) return;
    if (count > static_cast<std::int64_t>(max_tokens)) count = static_cast<std::int64_t>(max_tokens);
    const std::int64_t block = start / kKv8Block + blockIdx.x;
    const std::int64_t base = block * kKv8Block;   // first token of the block
    if (base >= start + count || block > 0x7fffffff / static_cast<std::int64_t>(kKv8Block)) return;
    const Kv8Byte* const rec = kv8_record(g, tables + static_cast<std::uint64_t>(seq) * g.max_pages, layer + l, head,
                                          static_cast<std::uint32_t>(block));
    if (rec == nullptr) return;
    const bool value = threadIdx.x >= D;
    const unsigned part = value ? threadIdx.x - D : threadIdx.x;
    const unsigned token0 = part / (D / 4u) * 4u, dim = part % (D / 4u) * 4u;
    const std::uint64_t row0 = (static_cast<std::uint64_t>(l) * seqs + seq) * max_tokens;
    const std::uint64_t width = static_cast<std::uint64_t>(g.kv_heads) * D;
    float* const dst = value ? v : k;
    if (dst != nullptr) {
        const float scale = kv8_load<float>(rec + (value ? 4 : 0));
        std::uint32_t c[4];   // of K a token's four dims, of V a dim's four tokens
#pragma unroll
        for (unsigned i = 0; i < 4u; ++i) {
            c[i] = kv8_load<std::uint32_t>(
                rec + (value ? kv8_v_offset(D, token0, dim + i) : kv8_k_offset(D, token0 + i, dim)));
        }
#pragma unroll
        for (unsigned t = 0; t < 4u; ++t) {
            const std::int64_t at_token = base + token0 + t;
            if (at_token < start || at_token >= start + count) continue;
            float x[4];
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i) {
                x[i] = kv8_value<TYPE>(value ? c[i] >> (8u * t) : c[t] >> (8u * i)) * scale;
            }
            float* const to = dst + (row0 + static_cast<std::uint64_t>(at_token - start)) * width +
                              static_cast<std::uint64_t>(head) * D + dim;
            if (aligned) {
                *reinterpret_cast<float4*>(to) = make_float4(x[0], x[1], x[2], x[3]);
            } else {
#pragma unroll
                for (unsigned i = 0; i < 4u; ++i) to[i] = x[i];
            }
        }
    }
    if (weights && threadIdx.x < kKv8Block) {
        const std::int64_t t = base + threadIdx.x;
        if (t >= start && t < start + count) {
            weights[(row0 + static_cast<std::uint64_t>(t - start)) * g.kv_heads + head] =
                kv8_load<float>(rec + kKv8Weights + 4u * threadIdx.x);
        }
    }
}

// The weights alone: a thread per (token, KV head), the heads of a token
// side by side as they are stored.
__global__ __launch_bounds__(256) void kv8_read_weights_kernel(Kv8Geometry g, std::uint32_t seqs,
                                                               const std::int32_t* __restrict__ starts,
                                                               const std::int32_t* __restrict__ lengths,
                                                               const std::int32_t* __restrict__ tables,
                                                               std::uint32_t layer, std::uint64_t max_tokens,
                                                               float* __restrict__ weights) {
    const std::uint32_t seq = blockIdx.y % seqs, l = blockIdx.y / seqs;
    const std::uint64_t idx = static_cast<std::uint64_t>(blockIdx.x) * 256u + threadIdx.x;
    const std::uint64_t j = idx / g.kv_heads;
    const std::uint32_t head = static_cast<std::uint32_t>(idx % g.kv_heads);
    const std::int64_t start = starts ? starts[seq] : 0;
    const std::int64_t t = start + static_cast<std::int64_t>(j);
    if (j >= max_tokens || start < 0 || static_cast<std::int64_t>(j) >= lengths[seq] || t > 0x7fffffff) return;
    const Kv8Byte* const rec = kv8_record(g, tables + static_cast<std::uint64_t>(seq) * g.max_pages, layer + l, head,
                                          static_cast<std::uint32_t>(t / kKv8Block));
    if (rec == nullptr) return;
    weights[((static_cast<std::uint64_t>(l) * seqs + seq) * max_tokens + j) * g.kv_heads + head] =
        kv8_load<float>(rec + kKv8Weights + 4u * static_cast<std::uint32_t>(t % kKv8Block));
}

// ---- eviction ----------------------------------------------------------------

constexpr unsigned kSelectThreads = 1024;
constexpr unsigned kSelectBins = 2 * kSelectThreads;
constexpr std::uint32_t kSelectKeys = 16384;   // keys held in LDS; longer sequences are read again each pass

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
// The want-th largest key of the middle tokens is found from the top by 11, 11
// and 10 bits (a histogram of the next digit over the keys that agree so far);
// then one pass in token order writes the first keep_first, every larger key,
// as many equal ones as are still wanted (the lowest tokens) and the last
// keep_last.  One workgroup has nothing to overlap its waits with, so the keys
// are read once, into LDS, and digits and places are found with prefix sums:
// 1000 tokens to 500 in 7 us, 4096 to 1024 in 13 (16 by four bytes, whose
// first has few values and many additions to one bin), the rounds' barriers.
// Past kSelectKeys every round reads the weights again, 64 bytes of each block
// (131072 tokens to 2048, gathered too, in 404).
__global__ __launch_bounds__(kSelectThreads) void kv8_select_kernel(
    Kv8Geometry g, const std::int32_t* __restrict__ lengths, const std::int32_t* __restrict__ tables,
    std::uint32_t layer, std::uint32_t layers, std::uint32_t keep_first, std::uint32_t keep_last, std::uint32_t budget,
    std::uint64_t max_tokens, std::int32_t* __restrict__ kept) {
    constexpr unsigned kWaves = kSelectThreads / 64u;
    __shared__ std::uint32_t keys[kSelectKeys];
    __shared__ std::uint32_t bins[kSelectBins];
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
    const auto read_key = [&](std::uint32_t t) __attribute__((always_inline)) -> std::uint32_t {
        const Kv8Byte* const rec = kv8_record(g, table, layer + l, head, t / kKv8Block);
        return rec ? weight_key(kv8_load<float>(rec + kKv8Weights + 4u * (t % kKv8Block))) : 0u;
    };
    // The middle tokens are lo + i, i < count; more of them than are wanted.
    const std::uint32_t lo = keep_first, count = static_cast<std::uint32_t>(n - keep_last) - lo;
    const std::uint32_t want = budget - keep_first - keep_last;
    for (std::uint32_t i = tid; i < keep_first; i += kSelectThreads) out[i] = static_cast<std::int32_t>(i);
    for (std::uint32_t i = tid; i < keep_last; i += kSelectThreads) {
        out[budget - keep_last + i] = static_cast<std::int32_t>(lo + count + i);
    }
    if (want == 0u) return;
    const std::uint32_t in_lds = count < kSelectKeys ? count : kSelectKeys;
#pragma unroll 4
    for (std::uint32_t i = tid; i < in_lds; i += kSelectThreads) keys[i] = read_key(lo + i);
    const auto key_of = [&](std::uint32_t i) __attribute__((always_inline)) -> std::uint32_t {
        return i < kSelectKeys ? keys[i] : read_key(lo + i);
    };
    std::uint32_t prefix = 0u, left = want;
    for (int shift = 21;; shift = shift == 21 ? 10 : 0) {   // 11, 11 and 10 bits
        bins[2u * tid] = bins[2u * tid + 1u] = 0u;
        __syncthreads();
        for (std::uint32_t i = tid; i < count; i += kSelectThreads) {
            const std::uint32_t key = key_of(i);
            // Shifts of 32 are undefined: the first round takes every key.
            const bool agrees = shift == 21 || (shift == 10 ? key >> 21 == prefix >> 21 : key >> 10 == prefix >> 10);
            if (agrees) atomicAdd(&bins[(key >> shift) & (shift == 0 ? 1023u : 2047u)], 1u);
        }
        __syncthreads();
        // Thread t holds two bins from the top; sums of those above.
        const std::uint32_t at = kSelectBins - 1u - 2u * tid, high = bins[at], low = bins[at - 1u];
        const std::uint32_t upto = wave_sums(high + low);
        if (lane == 63u) wave_above[wave] = upto;
        __syncthreads();
        std::uint32_t before = upto - high - low;
#pragma unroll
        for (unsigned w = 0; w < kWaves; ++w) before += w < wave ? wave_above[w] : 0u;
        if (before < left && before + high + low >= left) {   // one thread: the left-th key is in one of its bins
            const bool upper = before + high >= left;
            found_prefix = prefix | (upper ? at : at - 1u) << shift;
            found_want = left - before - (upper ? 0u : high);
        }
        __syncthreads();
        prefix = found_prefix;
        left = found_want;
        if (shift == 0) break;
    }
    // prefix is the want-th largest key, left how many keys equal to it stay.
    // A thread's tokens lie together, so one prefix sum over the threads places
    // them (16384 tokens at a time: 16 a thread, whose weights are one line).
    std::uint32_t base_above = 0u, base_equal = 0u;   // larger and equal keys before these tokens
    for (std::uint32_t from = 0u; from < count; from += kSelectKeys) {
        const std::uint32_t here = count - from < kSelectKeys ? count - from : kSelectKeys;
        const std::uint32_t each = (here + kSelectThreads - 1u) / kSelectThreads;
        const std::uint32_t begin = from + (tid * each < here ? tid * each : here);
        const std::uint32_t end = from + here - begin < each ? from + here : begin + each;
        std::uint32_t above = 0u, equal = 0u;
        for (std::uint32_t i = begin; i < end; ++i) {
            const std::uint32_t key = key_of(i);
            above += key > prefix ? 1u : 0u;
            equal += key == prefix ? 1u : 0u;
        }
        const std::uint32_t above_upto = wave_sums(above), equal_upto = wave_sums(equal);
        if (lane == 63u) {
            wave_above[wave] = above_upto;
            wave_equal[wave] = equal_upto;
        }
        __syncthreads();
        std::uint32_t a = base_above + above_upto - above, e = base_equal + equal_upto - equal;
#pragma unroll
        for (unsigned w = 0; w < kWaves; ++w) {
            a += w < wave ? wave_above[w] : 0u;
            e += w < wave ? wave_equal[w] : 0u;
            base_above += wave_above[w];
            base_equal += wave_equal[w];
        }
        for (std::uint32_t i = begin; i < end; ++i) {
            const std::uint32_t key = key_of(i);
            if (key > prefix || (key == prefix && e < left)) {
                out[keep_first + a + (e < left ? e : left)] = static_cast<std::int32_t>(lo + i);
            }
            a += key > prefix ? 1u : 0u;
            e += key == prefix ? 1u : 0u;
        }
        __syncthreads();
    }
}

// Gathers the kept tokens of a (sequence, layer, KV head) into blocks of the
// new table.  A block's scale is the largest of its tokens' scales, so a
// block whose tokens come from one block keeps its codes, and others are
// rounded once.  Threads as in the append; a token's source, scale and the
// ratio its codes take are found once, by 16 threads for K and 16 for V.
// With a quarter of the tokens kept nearly every 64-byte piece of the old
// codes is touched: the old sequence is read whole (six layers of sequences
// of 900..4100 tokens, 63 MB, and 25 MB written, in 32 us).  Measured slower:
// four blocks a workgroup with their loads together (41 us), and 16 bytes a
// dim and old block with the tokens picked from registers (52 us) or from LDS
// (36 us); fewer workgroups a CU then cover each other's waits.
//
// B > 1: in place.  One workgroup takes all blocks in ascending order, B at a
// time.  Block b's tokens come from blocks >= b, so reading ahead is always
// safe, and a block may be written once every block up to it has been read:
// all B are read, with the sources of the next B looked up meanwhile, then
// written (24 sequences and layers of 4096 tokens to 1024, four KV heads, the
// whole call: 203 us with one block at a time and no reading ahead, 78 so; 38
// to another table).
template <int TYPE, unsigned D, unsigned B>
__global__ __launch_bounds__(2 * D * B) void kv8_compact_kernel(Kv8Geometry g, const std::int32_t* tables,
                                                                const std::int32_t* new_tables, std::uint32_t layer,
                                                                std::uint32_t layers, std::uint32_t budget,
                                                                std::uint32_t blocks, const std::int32_t* kept) {
#pragma clang fp contract(off)
    constexpr unsigned kBuffers = B > 1u ? 2u : 1u;
    struct Source {
        const unsigned char* record[kKv8Block];
        std::uint32_t slot[kKv8Block];
        float ratio[2][kKv8Block];                 // below zero: the code stays as it is
        float scale[2];
    };
    __shared__ Source sources[kBuffers][B];
    const std::uint32_t head = blockIdx.y % g.kv_heads, l = blockIdx.y / g.kv_heads, seq = blockIdx.z;
    const unsigned tid = threadIdx.x % (2u * D), sub = threadIdx.x / (2u * D);
    const bool value = tid >= D;
    const unsigned part = value ? tid - D : tid;
    const unsigned token = part / (D / 16u), chunk = part % (D / 16u);
    const std::int32_t* const table = tables + static_cast<std::uint64_t>(seq) * g.max_pages;
    const std::int32_t* const new_table = new_tables + static_cast<std::uint64_t>(seq) * g.max_pages;
    const std::int32_t* const list =
        kept + ((static_cast<std::uint64_t>(seq) * layers + l) * g.kv_heads + head) * budget;
    if (B > 1u && list[budget - 1u] < static_cast<std::int32_t>(budget)) return;   // everything stays where it is
    // Where the tokens of block b come from; the token's weight for K's thread.
    const auto look_up = [&](std::uint32_t b, Source& from) __attribute__((always_inline)) -> float {
        float weight = 0.0f;
        if (part < kKv8Block) {
            const std::uint64_t i = static_cast<std::uint64_t>(b) * kKv8Block + part;
            const std::int32_t t = i < budget ? list[i] : -1;
            const unsigned char* src = nullptr;
            float s = 0.0f;
            unsigned slot = 0u;
            if (t >= 0) {
                slot = static_cast<std::uint32_t>(t) % kKv8Block;
                src = (const unsigned char*)kv8_record(g, table, layer + l, head, static_cast<std::uint32_t>(t) / kKv8Block);
                if (src) {
                    s = reinterpret_cast<const float*>(src)[value ? 1 : 0];
                    weight = reinterpret_cast<const float*>(src + kKv8Weights)[slot];
                }
            }
            // Scales are not negative, so their bits order them, NaN on top:
            // a poisoned token poisons its new block.
            std::uint32_t top = __float_as_uint(s);
#pragma unroll
            for (int off = 8; off > 0; off >>= 1) {
                const std::uint32_t o = static_cast<std::uint32_t>(__shfl_xor(static_cast<int>(top), off));
                top = o > top ? o : top;
            }
            const float scale = __uint_as_float(top);
            if (!value) {
                from.record[part] = src;
                from.slot[part] = slot;
            }
            from.ratio[value ? 1 : 0][part] = s == scale ? -1.0f : scale > 0.0f ? s / scale : 0.0f;
            if (part == 0u) from.scale[value ? 1 : 0] = scale;
        }
        return weight;
    };
    unsigned turn = 0u;
    std::uint32_t b = blockIdx.x * B + sub;
    if (list[static_cast<std::uint64_t>(b - sub) * kKv8Block] < 0) return;   // no tokens from here on
    float weight = look_up(b, sources[0][sub]);
    for (;;) {
        const bool stored = B == 1u || (b < blocks && list[static_cast<std::uint64_t>(b) * kKv8Block] >= 0);
        unsigned char* const dst = stored ? (unsigned char*)kv8_record(g, new_table, layer + l, head, b) : nullptr;
        __syncthreads();
        const Source& from = sources[turn][sub];
        const float* const ratios = from.ratio[value ? 1 : 0];
        u32x4 codes;
        if (value) {
            std::uint32_t was[16];   // all asked for before the first is used
#pragma unroll
            for (unsigned i = 0; i < 16u; ++i) {
                was[i] = from.record[i] ? from.record[i][kv8_v_offset(D, from.slot[i], part)] : kv8_zero_code<TYPE>();
            }
#pragma unroll
            for (unsigned i = 0; i < 16u; ++i) {
                if (ratios[i] >= 0.0f) was[i] = kv8_recode<TYPE>(was[i], ratios[i]);
            }
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i) {
                codes[i] = was[4u * i] | was[4u * i + 1u] << 8 | was[4u * i + 2u] << 16 | was[4u * i + 3u] << 24;
            }
        } else if (from.record[token] != nullptr) {
            codes = *reinterpret_cast<const u32x4*>(from.record[token] + kv8_k_offset(D, from.slot[token], chunk * 16u));
            const float ratio = ratios[token];
            if (ratio >= 0.0f) {
#pragma unroll
                for (unsigned i = 0; i < 16u; ++i) {
                    const std::uint32_t was = (codes[i >> 2] >> (8u * (i & 3u))) & 0xffu;
                    codes[i >> 2] = (codes[i >> 2] & ~(0xffu << (8u * (i & 3u)))) |
                                    kv8_recode<TYPE>(was, ratio) << (8u * (i & 3u));
                }
            }
        } else {
#pragma unroll
            for (unsigned i = 0; i < 4u; ++i) codes[i] = kv8_zero_code<TYPE>() * 0x01010101u;
        }
        const float scale = from.scale[value ? 1 : 0];
        const std::uint32_t next = b + B;
        const bool more = B > 1u && next - sub < blocks && list[static_cast<std::uint64_t>(next - sub) * kKv8Block] >= 0;
        float next_weight = 0.0f;
        if (more) next_weight = look_up(next, sources[kBuffers - 1u - turn][sub]);
        if (B > 1u) __syncthreads();   // the blocks' tokens are read: what they share with them may go
        if (dst != nullptr) {
            const unsigned at = value ? kv8_v_offset(D, 0u, part) : kv8_k_offset(D, token, chunk * 16u);
            *reinterpret_cast<u32x4*>(dst + at) = codes;
            if (part == 0u) reinterpret_cast<float*>(dst)[value ? 1 : 0] = scale;
            if (tid < kKv8Block) reinterpret_cast<float*>(dst + kKv8Weights)[tid] = weight;
        }
        if (!more) return;
        b = next;
        weight = next_weight;
        turn = kBuffers - 1u - turn;
    }
}

} // namespace

hipError_t launch_kv8_append(const Kv8Geometry& g, const float* qkv, std::uint64_t stride, std::uint64_t q_width,
                             std::uint32_t m, const std::int32_t* positions, const std::int32_t* tables,
                             std::uint32_t layer, hipStream_t stream) {
    const dim3 grid(m, g.kv_heads);
    const bool aligned = reinterpret_cast<std::uintptr_t>(qkv) % 16u == 0 && stride % 4u == 0 && q_width % 4u == 0;
#define AIR_KV8_APPEND(T, D)                                                                                     \
    hipLaunchKernelGGL((kv8_append_kernel<T, D>), grid, dim3(2 * D), 0, stream, g, qkv, stride, q_width, m, positions, \
                       tables, layer, aligned)
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
    if (!k && !v) {
        const std::uint64_t threads = max_tokens * g.kv_heads;
        hipLaunchKernelGGL(kv8_read_weights_kernel, dim3(static_cast<unsigned>((threads + 255u) / 256u), seqs * layers),
                           dim3(256), 0, stream, g, seqs, starts, lengths, tables, layer, max_tokens, weights);
        return hipGetLastError();
    }
    // A start inside a block makes the tokens span one more.
    const std::uint64_t blocks = (max_tokens + kKv8Block - 1u) / kKv8Block + (starts ? 1u : 0u);
    const dim3 grid(static_cast<unsigned>(blocks), g.kv_heads, seqs * layers);
    const bool aligned = reinterpret_cast<std::uintptr_t>(k) % 16u == 0 && reinterpret_cast<std::uintptr_t>(v) % 16u == 0;
#define AIR_KV8_READ(T, D)                                                                                           \
    hipLaunchKernelGGL((kv8_read_kernel<T, D>), grid, dim3(2 * D), 0, stream, g, seqs, starts, lengths, tables, layer, \
                       max_tokens, k, v, weights, aligned)
    if (g.type == kKv8I8) {
        if (g.head_dim == 128u) AIR_KV8_READ(kKv8I8, 128);
        else AIR_KV8_READ(kKv8I8, 64);
    } else {
        if (g.head_dim == 128u) AIR_KV8_READ(kKv8E4M3, 128);
        else AIR_KV8_READ(kKv8E4M3, 64);
    }
#undef AIR_KV8_READ
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
#define AIR_KV8_COMPACT_BLOCKS(T, D, B)                                                                              \
    hipLaunchKernelGGL((kv8_compact_kernel<T, D, B>), grid, dim3(2 * D * B), 0, stream, g, tables, new_tables, layer, \
                       layers, budget, blocks, kept)
#define AIR_KV8_COMPACT(T, D)                                    \
    do {                                                         \
        if (in_place) AIR_KV8_COMPACT_BLOCKS(T, D, 512 / D);     \
        else AIR_KV8_COMPACT_BLOCKS(T, D, 1);                    \
    } while (false)
    if (g.type == kKv8I8) {
        if (g.head_dim == 128u) AIR_KV8_COMPACT(kKv8I8, 128);
        else AIR_KV8_COMPACT(kKv8I8, 64);
    } else {
        if (g.head_dim == 128u) AIR_KV8_COMPACT(kKv8E4M3, 128);
        else AIR_KV8_COMPACT(kKv8E4M3, 64);
    }
#undef AIR_KV8_COMPACT
#undef AIR_KV8_COMPACT_BLOCKS
    return hipGetLastError();
}

} // namespace air_hip

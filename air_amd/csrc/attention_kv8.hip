// attention_kv8.hip -- attention over the paged 8-bit KV cache, and the
// attention weights it gathers.
//
//   s_t = (q . k_t) / sqrt(D),  p_t = e^(s_t - m) / sum e^(s - m),
//   out = sum_t p_t v_t,        weight_t (+)= sum over rows and q heads of p_t
//
// Codes are exact in f16, and an f32 operand is the sum of two f16 values to
// 22 bits (its rounding and the rounding of what that leaves), so both
// products run on v_mfma_f32_16x16x32_f16 with two instructions where one
// f16 operand would take one: q = hi + lo against K codes, p = hi + lo
// against V codes, summed in f32.  The result differs from a float64
// attention over the same codes by 3e-7 to 6e-7 relative (torch's f32 products
// and softmax over the decoded values: 4e-7 to 2e-6); a single f16 p would
// leave 2e-4.
//
// A wave walks chunks of 64 tokens (four blocks) of one KV head for 16 query
// vectors, with nothing staged in LDS:
//
//   S^T = K Q^T   row i of tile b is token 4 b + i % 4 of block i / 4, so
//                 lane (vector, g) ends with all 16 tokens of block g, in
//                 order: one scale of K and of V a lane, and p lies as
//   O^T += V^T P^T  wants it, 8 tokens of block g in lane group g a step.
//
// So the record's K and V codes go from memory into operand registers, a
// vector's statistics stay in its lanes (lane % 16), and an output lane holds
// four consecutive dims of one vector.
//
// Running references are whole numbers, in powers of two: M >= every s log2(e)
// so far (for the denominator) and M2 >= every s log2(e) + log2(scale of V) (for
// the numerators, whose p carries V's scale: a block of large values does not
// take the low bits of the others).  Rescaling by a power of two is exact.  M
// is an f32, so that scores of any size up to f32's largest do; M2 is held as
// its lead over M.
//
// What bounds it.  Decode over a cache larger than the chip's: reading it (48
// rows over 4000..16000 tokens, 32 q heads on 8 KV heads of 128 dims: 191 us,
// 5.2 TB/s of the 985 MB, as a large copy).  Fewer tokens: the waits of one
// walk (32 rows over 500..1200 tokens: 11.5 us, 2.3 TB/s).  Prompts: the
// alternation of products and softmax.  Vector operations, some 20 a score, take
// a third of the wave time and so do the matrix cores, which multiply both
// halves of an operand; the two waves of a SIMD do the one and the other in
// phases that hardly overlap (602 rows over 3300..3801 tokens, 28 q heads: 85
// us, 345 TFLOP/s of the products' 29 GFLOP).
#include "air_hip_device.hpp"
#include "air_hip_kernels.hpp"
#include "air_hip_kv8.hpp"

namespace air_hip {
namespace {

constexpr unsigned kWaves = 4;             // waves of a workgroup, but for short decode steps
constexpr unsigned kThreads = 64 * kWaves;
constexpr unsigned kShortWaves = 8;
constexpr unsigned kVectors = 16;          // query vectors of an MFMA tile
constexpr unsigned kRunTiles = 2;          // MFMA tiles of a workgroup where runs have several rows
constexpr unsigned kChunkBlocks = 4;       // blocks of a chunk, one per lane group
constexpr unsigned kChunkTokens = kChunkBlocks * kKv8Block;
constexpr float kNone = -0x1.fffffep127f;  // a reference that no score has set: below all others
constexpr int kNone2 = -(1 << 29);         // the same of M2
constexpr int kPBits = 15;                 // p' < 2^15 in f16: the largest p' keeps 2^-38 of itself
constexpr unsigned kStat = 4;              // floats before a partial's D sums

// Codes of blocks without a page: any finite value will do under a mask.
__device__ __align__(16) unsigned char g_no_record[kKv8Codes + 2 * kKv8Block * 128];

// 16 code bytes as two f16 operands of eight.
template <int TYPE>
__device__ __forceinline__ void codes_to_half(const u32x4& c, half8v& a, half8v& b) {
    half2v h[8];
#pragma unroll
    for (unsigned i = 0; i < 4u; ++i) {
        if constexpr (TYPE == kKv8I8) {
            q8_dword_to_half(c[i], h[2u * i], h[2u * i + 1u]);
        } else {
            h[2u * i] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], 1.0f, false);
            h[2u * i + 1u] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], 1.0f, true);
        }
    }
#pragma unroll
    for (unsigned i = 0; i < 4u; ++i) {
        a[2u * i] = h[i][0];
        a[2u * i + 1u] = h[i][1];
        b[2u * i] = h[4u + i][0];
        b[2u * i + 1u] = h[4u + i][1];
    }
}

// x share = hi + lo to 22 bits, for two x.  hi passes an empty asm so that
// both halves go by one rounding of it: left to itself the compiler may round
// the product straight to f16 in one place and by way of f32 in the other,
// and next to a tie these differ (seen as single weights off by 2^-11).
__device__ __forceinline__ void split_products(float x0, float x1, float share, half2v& hi, half2v& lo) {
    typedef float float2v __attribute__((ext_vector_type(2)));
    std::uint32_t bits = __builtin_bit_cast(std::uint32_t, __builtin_convertvector(float2v{x0 * share, x1 * share}, half2v));
    asm("" : "+v"(bits));
    hi = __builtin_bit_cast(half2v, bits);
    lo[0] = static_cast<_Float16>(__builtin_fmaf(x0, share, -static_cast<float>(hi[0])));
    lo[1] = static_cast<_Float16>(__builtin_fmaf(x1, share, -static_cast<float>(hi[1])));
}

// The B operands of the products with K of one query vector (lane % 16), and
// the factor that undoes their power-of-two scale.  An MFMA adds its 32
// products in a window of 24 bits below the largest and drops what lies under
// it (the sum then meets the accumulator with one rounding), so hi is whole:
// with the vector's largest magnitude in [2^10, 2^11), hi times a code is a
// multiple of the code's last place and 32 of them fit the window.  lo is the
// f16 nearest to the rest, to 2^-24 of the largest magnitude.
template <unsigned D>
struct QueryFragments {
    half8v hi[D / 32], lo[D / 32];
    float undo;
};

template <unsigned D>
__device__ __forceinline__ void load_query(const float* q, unsigned grp, QueryFragments<D>& f) {
    float x[D / 4];
    float top = 0.0f;
#pragma unroll
    for (unsigned s = 0; s < D / 64u; ++s) {
#pragma unroll
        for (unsigned i = 0; i < 4u; ++i) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (q) v = *reinterpret_cast<const float4*>(q + 64u * s + 16u * grp + 4u * i);
            x[16u * s + 4u * i] = v.x;
            x[16u * s + 4u * i + 1u] = v.y;
            x[16u * s + 4u * i + 2u] = v.z;
            x[16u * s + 4u * i + 3u] = v.w;
        }
    }
#pragma unroll
    for (unsigned i = 0; i < D / 4u; ++i) top = fmaxf(top, fabsf(x[i]));
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;   // -127: zero or subnormal; 128: not finite
    e = e < -110 ? -110 : e > 127 ? 127 : e;   // both scales stay normal numbers
    const float scale = __uint_as_float(static_cast<std::uint32_t>(127 + 10 - e) << 23);
    f.undo = __uint_as_float(static_cast<std::uint32_t>(127 - 10 + e) << 23);
#pragma unroll
    for (unsigned i = 0; i < D / 32u; ++i) {
#pragma unroll
        for (unsigned j = 0; j < 8u; ++j) {
            const float y = x[8u * i + j] * scale, whole = rintf(y);
            f.hi[i][j] = static_cast<_Float16>(whole);
            f.lo[i][j] = static_cast<_Float16>(y - whole);
        }
    }
}

// A vector's operands, kept for the kernel that gathers weights: 16 bytes of
// lane group grp at (2 i + part) * 4 + grp, so that a load takes 64 bytes of a
// vector together.
template <unsigned D>
__device__ __forceinline__ void keep_query(half8v* at, unsigned grp, const QueryFragments<D>& f) {
#pragma unroll
    for (unsigned i = 0; i < D / 32u; ++i) {
        at[8u * i + grp] = f.lo[i];
        at[8u * i + 4u + grp] = f.hi[i];
    }
}
template <unsigned D>
__device__ __forceinline__ void kept_query(const half8v* at, unsigned grp, QueryFragments<D>& f) {
#pragma unroll
    for (unsigned i = 0; i < D / 32u; ++i) {
        f.lo[i] = at[8u * i + grp];
        f.hi[i] = at[8u * i + 4u + grp];
    }
}

// A lane's codes of the chunk's K: tile b, 64-dim step s.
template <unsigned D>
struct KeyCodes {
    u32x4 c[4][D / 64];
};

template <unsigned D>
__device__ __forceinline__ void load_keys(const Kv8Byte* rec, unsigned lane, KeyCodes<D>& k) {
    const Kv8Byte* const at = rec + kKv8Codes + (lane >> 4) * 64u + (lane & 3u) * 16u;
#pragma unroll
    for (unsigned b = 0; b < 4u; ++b) {
#pragma unroll
        for (unsigned s = 0; s < D / 64u; ++s) {
            k.c[b][s] = kv8_load<u32x4>(at + b * (D * 4u) + s * 256u);
        }
    }
}

// What a block's scores are multiplied by.  Scores are whole numbers below
// 2^27, so a factor below f32's normal range leaves nothing of them (nor does
// a scale of zero, whose codes are zero): the smallest normal number stands
// for it, which keeps masked scores at -inf where zero would make them NaN.
// A NaN scale passes.
constexpr float kLeastFactor = 0x1p-126f;
__device__ __forceinline__ float score_factor(float unit, float k_scale) {
    const float f = unit * k_scale;
    return f < kLeastFactor ? kLeastFactor : f;
}

// Scores that may pass 2^23 are multiplied by their factor first, rounded to
// f32, whose neighbours are one and more apart there: only so is the largest of
// them its own reference, and its 2^(s - M) 1.  Below, the product is exact
// until M is taken off it.  Every kernel decides by the factor alone, so all of
// them take the same scores.  Returns whether a lane's block was one.
template <int TYPE, unsigned D>
__device__ __forceinline__ bool round_large(float4v (&s)[4], float& factor) {
    constexpr float kLargest = static_cast<float>(D) * (TYPE == kKv8I8 ? 127.0f : 448.0f) * 0x1p11f;
    const bool large = factor >= 0x1p23f / kLargest;
    if (__builtin_expect(!__any(large), 1)) return false;
#pragma unroll
    for (unsigned b = 0; b < 4u; ++b) {
#pragma unroll
        for (unsigned r = 0; r < 4u; ++r) s[b][r] = large ? s[b][r] * factor : s[b][r];
    }
    factor = large ? 1.0f : factor;
    return true;
}
// 2^(score * factor - base), one rounding
__device__ __forceinline__ float score_power(float score, float factor, float base) {
    return __builtin_amdgcn_exp2f(__builtin_fmaf(score, factor, -base));
}

// A lane's codes of the chunk's V: dim 16 t + lane % 16 of block lane / 16.
template <unsigned D>
__device__ __forceinline__ void load_values(const Kv8Byte* rec, unsigned lane, u32x4 (&v)[D / 16]) {
    const Kv8Byte* const at = rec + kKv8Codes + kKv8Block * D + (lane & 15u) * 16u;
#pragma unroll
    for (unsigned t = 0; t < D / 16u; ++t) v[t] = kv8_load<u32x4>(at + t * 256u);
}

// The two scales of a record.
__device__ __forceinline__ float2 load_scales(const Kv8Byte* rec) {
    const u32x2 v = kv8_load<u32x2>(rec);
    return make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
}

// S^T of the chunk: score[b][r] is token 4 b + r of this lane's block for
// vector lane % 16, times the fragments' scale.
// The low parts come first: their roundings are those of a small sum.
template <int TYPE, unsigned D>
__device__ __forceinline__ void chunk_scores(const KeyCodes<D>& k, const QueryFragments<D>& q, float4v (&score)[4]) {
#pragma unroll
    for (unsigned b = 0; b < 4u; ++b) {
        half8v a[D / 32];
        score[b] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (unsigned s = 0; s < D / 64u; ++s) codes_to_half<TYPE>(k.c[b][s], a[2u * s], a[2u * s + 1u]);
#pragma unroll
        for (unsigned i = 0; i < D / 16u; ++i) {
            const half8v f = i < D / 32u ? q.lo[i] : q.hi[i - D / 32u];
            score[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i % (D / 32u)], f, score[b], 0, 0, 0);
        }
    }
}

// max over the four lane groups of a vector, in every lane of it.
template <typename T>
__device__ __forceinline__ T groups_max(T x) {
    const auto swapped = [](const auto& pair, unsigned i) { return __builtin_bit_cast(T, static_cast<std::uint32_t>(pair[i])); };
    const std::uint32_t bits = __builtin_bit_cast(std::uint32_t, x);
    const auto h = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
    const T a = swapped(h, 0u), b = swapped(h, 1u), m = a > b ? a : b;
    const std::uint32_t half = __builtin_bit_cast(std::uint32_t, m);
    const auto q = __builtin_amdgcn_permlane16_swap(half, half, false, false);
    const T c = swapped(q, 0u), d = swapped(q, 1u);
    return c > d ? c : d;
}

// The difference of two references as an exponent: what is past 2^28 either
// way leaves nothing of an f32, and sums of a few such stay in 32 bits.
__device__ __forceinline__ int powers(float difference) {
    return static_cast<int>(__builtin_amdgcn_fmed3f(difference, -0x1p28f, 0x1p28f));
}

// The scores of a chunk into p' = hi + lo, the B operands of the products
// with V, and into the denominator.  `ahead`: how far this lane's vector lies
// behind the block's first token (it sees tokens 0..ahead); `here`: the block
// has a page; scale: of K and V; `far`: whether a chunk of the wave's had
// scores that may pass 2^23.
template <int TYPE, unsigned D>
__device__ __forceinline__ void soften(float4v (&s)[4], float unit, float2 scale, bool here, int ahead, float& ref, int& ref2,
                                       bool& far, float& l, float4v (&o)[D / 16], half8v (&p_hi)[2], half8v (&p_lo)[2]) {
    float factor = score_factor(unit, scale.x);
    float v_scale = scale.y;
    const int exponent = __builtin_amdgcn_frexp_expf(v_scale);   // scale of V < 2^exponent
    if (!__all(here && ahead >= 15)) {
        // What a vector does not see scores -inf; a block that it sees
        // nothing of has no scales either (they may be NaN).
        const int limit = here ? ahead : -1;
        factor = limit < 0 ? kLeastFactor : factor;
        v_scale = limit < 0 ? 0.0f : v_scale;
#pragma unroll
        for (unsigned b = 0; b < 4u; ++b) {
#pragma unroll
            for (unsigned r = 0; r < 4u; ++r) {
                s[b][r] = static_cast<int>(4u * b + r) <= limit ? s[b][r] : -__builtin_huge_valf();
            }
        }
    }
    far |= round_large<TYPE, D>(s, factor);
    float top = s[0][0];
#pragma unroll
    for (unsigned b = 0; b < 4u; ++b) {
#pragma unroll
        for (unsigned r = 0; r < 4u; ++r) top = fmaxf(top, s[b][r]);
    }
    // The block's own references; the vector's only move when one of its
    // blocks passes them.
    const float block_m = ceilf(top * factor);
    const int held_m = powers(ref);
    int block_m2 = powers(far ? block_m - ref : block_m) + exponent;
    if (__builtin_expect(far, 0)) block_m2 += held_m;
    block_m2 = v_scale == 0.0f ? kNone2 : block_m2;
    if (__any(block_m > ref || block_m2 > ref2)) {
        const float next = groups_max(block_m > ref ? block_m : ref);
        const int down = powers(ref - next);
        int next2, down2;
        if (__builtin_expect(far, 0)) {            // by way of the leads, whatever M is
            const int held = ref2 - held_m + down > kNone2 ? ref2 - held_m + down : kNone2;
            const int mine = v_scale == 0.0f ? kNone2 : powers(block_m - next) + exponent;
            const int lead = groups_max(mine > held ? mine : held);
            down2 = held - lead;
            next2 = powers(next) + lead;
        } else {
            next2 = groups_max(block_m2 > ref2 ? block_m2 : ref2);
            down2 = ref2 - next2;
        }
        l = __builtin_amdgcn_ldexpf(l, down);
#pragma unroll
        for (unsigned t = 0; t < D / 16u; ++t) {
#pragma unroll
            for (unsigned r = 0; r < 4u; ++r) o[t][r] = __builtin_amdgcn_ldexpf(o[t][r], down2);
        }
        ref = next;
        ref2 = next2;
    }
    // p' = 2^(s - base) * share, below 2^kPBits; a scale of V far below the
    // others' (or zero) keeps base near M, so the same powers also sum up the
    // denominator.  s - base is small where p is large, and rounded once.
    const int lead = ref2 - powers(ref);
    int e = lead - 40;
    e = v_scale == 0.0f || exponent < e ? e : exponent;
    int over = lead - e, up = kPBits - e;          // base - M, and the exponent of share / (scale of V)
    const float base = ref + static_cast<float>(over);
    if (__builtin_expect(far, 0)) {
        // Past 2^24 the sum was rounded, so the exponents follow from what it
        // became; p' is as large as before, so where share would overflow the
        // power is zero.
        over = powers(base - ref);
        up = kPBits - lead + over;
        up = up < 100 - exponent ? up : 100 - exponent;
    }
    const float share = __builtin_amdgcn_ldexpf(v_scale, up);
    float sum = 0.0f;
#pragma unroll
    for (unsigned b = 0; b < 4u; ++b) {
#pragma unroll
        for (unsigned r = 0; r < 4u; r += 2u) {
            const float x0 = score_power(s[b][r], factor, base);
            const float x1 = score_power(s[b][r + 1u], factor, base);
            sum += x0;
            sum += x1;
            half2v hi, lo;
            split_products(x0, x1, share, hi, lo);
            p_hi[b >> 1][4u * (b & 1u) + r] = hi[0];
            p_hi[b >> 1][4u * (b & 1u) + r + 1u] = hi[1];
            p_lo[b >> 1][4u * (b & 1u) + r] = lo[0];
            p_lo[b >> 1][4u * (b & 1u) + r + 1u] = lo[1];
        }
    }
    l += __builtin_amdgcn_ldexpf(sum, over);
}

// The rows of a tile: with RUNS up to tile_rows rows of one run (as many whole
// groups of q heads as fit its 16 NV vectors, at least one), otherwise one row.  A group of more than 16 NV q heads is cut into parts.
struct Tile {
    std::uint32_t row, rows;       // first row, rows (0: no tile)
    std::uint32_t head, heads;     // q heads of each row
};

// The tile that is `index`-th to start, of at most `tiles` tiles of the runs;
// they count down, as the last rows of a run reach furthest.
__device__ __forceinline__ Tile find_tile(std::uint32_t index, std::uint32_t tiles, const std::int32_t* __restrict__ run_starts,
                                          std::uint32_t runs, std::uint32_t m, std::uint32_t tile_rows) {
    const unsigned lane = threadIdx.x & 63u;
    std::uint32_t run, first;                      // the tile's run, and that run's first tile
    std::int64_t begin, end;
    if (runs <= 64u) {
        // The runs' tiles one after the other, so that the empty ones come last:
        // spread between the others they leave some CUs two tiles and others
        // none (24 runs of 4 rows of 28 q heads over 3000 tokens: 43 us, 30 so).
        const std::int32_t b = lane < runs ? run_starts[lane] : 0, e = lane < runs ? run_starts[lane + 1u] : 0;
        const bool held = b >= 0 && e > b && static_cast<std::uint32_t>(e) <= m;
        const std::uint32_t mine = held ? (static_cast<std::uint32_t>(e - b) + tile_rows - 1u) / tile_rows : 0u;
        const std::uint32_t upto = wave_sums(mine);
        const std::uint32_t all = __builtin_amdgcn_readlane(upto, 63);
        if (index >= all) return Tile{0u, 0u, 0u, 0u};
        index = all - 1u - index;
        run = static_cast<std::uint32_t>(__builtin_ctzll(__ballot(upto > index)));
        first = __builtin_amdgcn_readlane(upto - mine, run);
        begin = static_cast<std::int32_t>(__builtin_amdgcn_readlane(b, run));
        end = static_cast<std::int32_t>(__builtin_amdgcn_readlane(e, run));
    } else {
        // Run i owns tiles run_starts[i] / tile_rows + i and on: at least as
        // many as its rows need, and the count over all runs needs no prefix
        // sum.  The wave looks 64 runs up at a time.
        index = tiles - 1u - index;
        std::uint32_t lo = 0u, hi = runs;          // the run is in [lo, hi)
        const auto first_tile = [&](std::uint32_t i) __attribute__((always_inline)) {
            const std::int32_t s = run_starts[i];
            return (s > 0 ? static_cast<std::uint32_t>(s) / tile_rows : 0u) + i;
        };
        while (hi - lo > 1u) {
            const std::uint32_t step = (hi - lo + 63u) / 64u;
            const std::uint32_t i = lo + lane * step;
            const bool below = i < hi && first_tile(i) <= index;
            const std::uint64_t mask = __ballot(below);
            if (mask == 0u) return Tile{0u, 0u, 0u, 0u};
            const std::uint32_t last = 63u - static_cast<std::uint32_t>(__builtin_clzll(mask));
            lo += last * step;
            hi = lo + step < hi ? lo + step : hi;
        }
        run = lo;
        first = first_tile(lo);
        begin = run_starts[lo];
        end = run_starts[lo + 1u];
        if (begin < 0 || end > static_cast<std::int64_t>(m) || first > index) return Tile{0u, 0u, 0u, 0u};
    }
    const std::int64_t row = begin + static_cast<std::int64_t>(index - first) * tile_rows;
    if (row >= end) return Tile{0u, 0u, 0u, 0u};
    const std::int64_t left = end - row;
    return Tile{static_cast<std::uint32_t>(row), static_cast<std::uint32_t>(left < tile_rows ? left : tile_rows), 0u, 0u};
}

// The (tile, heads) pairs of a launch, one workgroup for each of the first
// `whole` ones and `splits` of split_chunks chunks for each of the others.
struct Kv8Work {
    std::uint32_t pair, tile, tile_head, split, split_chunks;
};
__device__ __forceinline__ Kv8Work kv8_work(const Kv8Cut& cut, std::uint32_t block, std::uint32_t tile_heads) {
    std::uint32_t pair = block, split = 0u, chunks = 0x7fffffffu / kChunkTokens;   // more than any tile has
    if (block >= cut.whole) {
        const std::uint32_t pairs = cut.pairs - cut.whole;
        pair = cut.whole + (block - cut.whole) % pairs;
        split = (block - cut.whole) / pairs;
        chunks = cut.split_chunks;
    }
    return Kv8Work{pair, pair / tile_heads, pair % tile_heads, split, chunks};
}

// A tile of up to 16 NV query vectors of one KV head per workgroup; its W waves
// take the chunks of its split in turn, every wave for all vectors, and meet
// at the end.  With NV > 1 the vectors' operands lie in LDS, and a chunk's
// codes are turned into f16 once for all of them: with 16 vectors a wave the
// conversions alone are up to 16 operations a score (602 rows over 3300..3801
// tokens: 208 us with 16 vectors and references moved in every chunk, 108 with
// 32 and moved when passed, 85 with what followed).  Measured slower there: 128
// vectors a workgroup whose waves share codes converted in LDS (98 us where
// this took 94), and 32x32x16 products (92 where this took 87): the waves wait
// longer between the phases, which they do not overlap, than fewer instructions
// save.
template <int TYPE, unsigned D, unsigned NV, bool RUNS, unsigned W>
__global__ __launch_bounds__(64 * W, NV == 1u && W == kWaves ? 3 : 2) void kv8_attention_kernel(
    Kv8Geometry g, const float* __restrict__ qkv, std::uint64_t stride, std::uint32_t m,
    const std::int32_t* __restrict__ positions, const std::int32_t* __restrict__ tables, std::uint32_t layer,
    std::uint32_t q_heads, const std::int32_t* __restrict__ run_starts, std::uint32_t runs, std::uint32_t tile_rows,
    std::uint64_t max_tokens, Kv8Cut cut, float score_scale, float* __restrict__ partials, float2* __restrict__ stats,
    half8v* __restrict__ queries, float* __restrict__ undos, float* __restrict__ out) {
    constexpr unsigned LD = D + 4;
    constexpr unsigned kTile = kVectors * NV;
    constexpr unsigned kFrags = D / 32;            // k steps of a score
    union Shared {
        half8v query[NV > 1u ? NV : 1u][kFrags][2][64];
        float sums[W][kTile][LD];
    };
    __shared__ Shared sh;
    __shared__ float undo_of[kTile];
    __shared__ float wave_m[W][kTile], wave_l[W][kTile];
    __shared__ int wave_power[W][kTile], wave_m2[W][kTile];
    const unsigned tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, grp = lane >> 4, col = lane & 15u;
    const std::uint32_t group = q_heads / g.kv_heads, parts = (group + kTile - 1u) / kTile;
    const Kv8Work work = kv8_work(cut, blockIdx.x, g.kv_heads * parts);
    const std::uint32_t split = work.split, split_chunks = work.split_chunks;
    const std::uint32_t kvh = work.tile_head / parts, part = work.tile_head % parts;
    Tile tile{work.tile, 1u, 0u, 0u};
    if constexpr (RUNS) tile = find_tile(work.tile, cut.pairs / (g.kv_heads * parts), run_starts, runs, m, tile_rows);
    if (tile.rows == 0u) return;
    tile.head = kvh * group + part * kTile;
    tile.heads = group - part * kTile < kTile ? group - part * kTile : kTile;
    const unsigned nq = tile.rows * tile.heads;

    // The furthest position of the tile, and those of this lane's vectors
    // (places without a vector go along with the furthest).
    const int most = static_cast<int>(max_tokens) - 1;
    int reach = -1;
    for (unsigned r = 0; r < tile.rows; ++r) {
        const int p = positions[tile.row + r];
        reach = p > reach ? p : reach;
    }
    reach = reach < most ? reach : most;
    int pos[NV];
#pragma unroll
    for (unsigned n = 0; n < NV; ++n) {
        const unsigned v = n * kVectors + col;
        pos[n] = v < nq ? positions[tile.row + v / tile.heads] : reach;
        pos[n] = pos[n] < reach ? pos[n] : reach;
    }
    const std::uint32_t chunks = reach < 0 ? 0u : static_cast<std::uint32_t>(reach) / kChunkTokens + 1u;
    const std::uint32_t live = chunks == 0u ? 1u : (chunks + split_chunks - 1u) / split_chunks;
    if (split >= live) return;
    const std::int32_t* const table = tables + static_cast<std::uint64_t>(tile.row) * g.max_pages;
    const std::uint32_t end = chunks < (split + 1u) * split_chunks ? chunks : (split + 1u) * split_chunks;

    const auto vector_at = [&](unsigned v) __attribute__((always_inline)) -> const float* {
        if (v >= nq) return nullptr;
        return qkv + static_cast<std::uint64_t>(tile.row + v / tile.heads) * stride +
               static_cast<std::uint64_t>(tile.head + v % tile.heads) * D;
    };
    QueryFragments<D> q;
    float undo[NV];
    if constexpr (NV == 1u) {
        load_query<D>(vector_at(col), grp, q);
        undo[0] = q.undo;
    } else {
        for (unsigned n = wave; n < NV; n += W) {
            load_query<D>(vector_at(n * kVectors + col), grp, q);
#pragma unroll
            for (unsigned i = 0; i < kFrags; ++i) {
                sh.query[n][i][0][lane] = q.lo[i];
                sh.query[n][i][1][lane] = q.hi[i];
            }
            const unsigned v = n * kVectors + col;
            if (grp == 0u) undo_of[v] = q.undo;
            if (queries && split == 0u && v < nq) {   // for the weights
                const std::uint64_t vector =
                    static_cast<std::uint64_t>(tile.row + v / tile.heads) * q_heads + tile.head + v % tile.heads;
                keep_query<D>(queries + vector * (D / 4u), grp, q);
                if (grp == 0u) undos[vector] = q.undo;
            }
        }
        __syncthreads();
#pragma unroll
        for (unsigned n = 0; n < NV; ++n) undo[n] = undo_of[n * kVectors + col];
    }

    float ref[NV], l[NV];                          // M and the denominator
    int ref2[NV];                                  // M2, as powers(M) and its lead
    bool far = false;
    float4v o[NV][D / 16];
#pragma unroll
    for (unsigned n = 0; n < NV; ++n) {
        ref[n] = kNone;
        ref2[n] = kNone2;
        l[n] = 0.0f;
#pragma unroll
        for (unsigned t = 0; t < D / 16u; ++t) o[n][t] = float4v{0.f, 0.f, 0.f, 0.f};
    }

    // Page ids are read a chunk ahead, before this chunk's codes: loads return
    // in order, so what waits for the ids does not wait for the codes.
    const Kv8Byte* const none = (const Kv8Byte*)g_no_record;
    const std::uint32_t from = split * split_chunks + wave;
    const auto page_of = [&](std::uint32_t block, std::uint32_t& slot) __attribute__((always_inline)) -> std::int32_t {
        slot = kv8_slot(g, block);
        return slot < g.max_pages ? table[slot] : -1;
    };
    // Pages of the blocks whose K and V this lane loads.
    std::uint32_t k_block = from * kChunkBlocks + (col >> 2), v_block = from * kChunkBlocks + grp, k_slot, v_slot;
    std::int32_t k_page = page_of(k_block, k_slot), v_page = page_of(v_block, v_slot);
    for (std::uint32_t c = from; c < end; c += W) {
        const Kv8Byte* const krec = kv8_record_in(g, k_page, k_slot, layer, kvh, k_block);
        const Kv8Byte* const vrec = kv8_record_in(g, v_page, v_slot, layer, kvh, v_block);
        const bool here = vrec != nullptr;
        k_block += W * kChunkBlocks;
        v_block += W * kChunkBlocks;
        k_page = page_of(k_block, k_slot);
        v_page = page_of(v_block, v_slot);
        KeyCodes<D> keys;
        u32x4 vals[D / 16];
        load_keys<D>(krec ? krec : none, lane, keys);
        const float2 now = load_scales(vrec ? vrec : none);
        load_values<D>(vrec ? vrec : none, lane, vals);
        float4v s[NV][4];
        if constexpr (NV == 1u) {
            chunk_scores<TYPE, D>(keys, q, s[0]);
        } else {
            asm volatile("" ::: "memory");         // the query operands are read again, not kept in registers
#pragma unroll
            for (unsigned b = 0; b < 4u; ++b) {
                half8v a[kFrags];
#pragma unroll
                for (unsigned i = 0; i < kFrags / 2u; ++i) codes_to_half<TYPE>(keys.c[b][i], a[2u * i], a[2u * i + 1u]);
#pragma unroll
                for (unsigned n = 0; n < NV; ++n) {
                    s[n][b] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (unsigned i = 0; i < 2u * kFrags; ++i) {   // low parts first
                        s[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i % kFrags], sh.query[n][i % kFrags][i / kFrags][lane],
                                                                         s[n][b], 0, 0, 0);
                    }
                }
            }
        }
        // Tokens of this lane's block that its vectors may attend to.
        const int first = static_cast<int>((c * kChunkBlocks + grp) * kKv8Block);
        half8v p_hi[NV][2], p_lo[NV][2];
#pragma unroll
        for (unsigned n = 0; n < NV; ++n) {
            soften<TYPE, D>(s[n], undo[n] * score_scale, now, here, pos[n] - first, ref[n], ref2[n], far, l[n], o[n], p_hi[n],
                            p_lo[n]);
        }
        if constexpr (TYPE == kKv8E4M3) {
            // Slots behind the tile's last token may hold NaN codes, which a
            // zero p does not silence.
            const int ahead = here ? reach - first : -1;
            if (__any(ahead < 15)) {
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const int bytes = ahead + 1 - 4 * w;
                    const std::uint32_t mask = bytes >= 4 ? 0xffffffffu : bytes <= 0 ? 0u : (1u << (8 * bytes)) - 1u;
#pragma unroll
                    for (unsigned t = 0; t < D / 16u; ++t) vals[t][w] &= mask;
                }
            }
        }
#pragma unroll
        for (unsigned t = 0; t < D / 16u; ++t) {
            half8v a[2];
            codes_to_half<TYPE>(vals[t], a[0], a[1]);
#pragma unroll
            for (unsigned n = 0; n < NV; ++n) {
                // One accumulator's products in a row: an MFMA takes 19.5
                // cycles so, 22.6 with two accumulators in turn, 26 with four.
#pragma unroll
                for (unsigned i = 0; i < 4u; ++i) {
                    const half8v f = i < 2u ? p_lo[n][i] : p_hi[n][i - 2u];
                    o[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i & 1u], f, o[n][t], 0, 0, 0);
                }
            }
        }
    }

    // The waves meet: sums in units of 2^(M + lead - kPBits), l of 2^M.
    if constexpr (NV > 1u) __syncthreads();        // the query operands make room
#pragma unroll
    for (unsigned n = 0; n < NV; ++n) {
        const unsigned v = n * kVectors + col;
        l[n] += __shfl_xor(l[n], 16);
        l[n] += __shfl_xor(l[n], 32);
        if (grp == 0u) {
            wave_m[wave][v] = ref[n];
            wave_power[wave][v] = powers(ref[n]);
            wave_m2[wave][v] = ref2[n];
            wave_l[wave][v] = l[n];
        }
#pragma unroll
        for (unsigned t = 0; t < D / 16u; ++t) *reinterpret_cast<float4v*>(&sh.sums[wave][v][16u * t + 4u * grp]) = o[n][t];
    }
    __syncthreads();
    for (unsigned idx = tid; idx < nq * (D / 4u); idx += 64u * W) {
        const unsigned v = idx / (D / 4u), d4 = idx % (D / 4u);
        float4v sums[W];
        float denominators[W];
        int power[W], m2[W], most_m = -(1 << 28), most_m2 = kNone2;
#pragma unroll
        for (unsigned w = 0; w < W; ++w) {
            power[w] = wave_power[w][v];
            m2[w] = wave_m2[w][v];
            denominators[w] = wave_l[w][v];
            sums[w] = *reinterpret_cast<const float4v*>(&sh.sums[w][v][4u * d4]);
        }
#pragma unroll
        for (unsigned w = 0; w < W; ++w) {
            most_m = power[w] > most_m ? power[w] : most_m;
            most_m2 = m2[w] > most_m2 ? m2[w] : most_m2;
        }
        float mm = static_cast<float>(most_m);
        int lead = most_m2 - most_m;
        if (__builtin_expect(most_m <= -(1 << 27) || most_m == 1 << 28, 0)) {
            // References too large for differences of their powers: the leads
            // stay, and M goes by its own differences.
            mm = kNone;
            for (unsigned w = 0; w < W; ++w) mm = wave_m[w][v] > mm ? wave_m[w][v] : mm;
            most_m = 0;
            most_m2 = kNone2;
#pragma unroll
            for (unsigned w = 0; w < W; ++w) {
                m2[w] -= power[w];
                power[w] = powers(wave_m[w][v] - mm);
                m2[w] += power[w];
                most_m2 = m2[w] > most_m2 ? m2[w] : most_m2;
            }
            lead = most_m2;
        }
        float total = 0.0f;
        float4v acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (unsigned w = 0; w < W; ++w) {
            total += __builtin_amdgcn_ldexpf(denominators[w], power[w] - most_m);
#pragma unroll
            for (unsigned r = 0; r < 4u; ++r) acc[r] += __builtin_amdgcn_ldexpf(sums[w][r], m2[w] - most_m2);
        }
        const std::uint64_t vector =
            static_cast<std::uint64_t>(tile.row + v / tile.heads) * q_heads + tile.head + v % tile.heads;
        if (live == 1u) {
            float4v y;
#pragma unroll
            for (unsigned r = 0; r < 4u; ++r) {
                y[r] = total == 0.0f ? 0.0f : __builtin_amdgcn_ldexpf(acc[r] / total, lead - kPBits);
            }
            *reinterpret_cast<float4v*>(out + vector * D + 4u * d4) = y;
            if (stats && d4 == 0u) stats[vector] = make_float2(mm, total == 0.0f ? 0.0f : 1.0f / total);
        } else {
            const std::uint64_t place = RUNS ? static_cast<std::uint64_t>(work.pair - cut.whole) * kTile + v : vector;
            float* const p = partials + (place * cut.splits + split) * (D + kStat);
            if (d4 == 0u) *reinterpret_cast<float4v*>(p) = float4v{mm, __int_as_float(lead), total, 0.0f};
            *reinterpret_cast<float4v*>(p + kStat + 4u * d4) = acc;
        }
    }
}

// Splits that a tile reaching to `reach` was cut into.
__device__ __forceinline__ std::uint32_t live_splits(int reach, std::uint64_t max_tokens, std::uint32_t split_chunks) {
    const int most = static_cast<int>(max_tokens) - 1;
    reach = reach < most ? reach : most;
    const std::uint32_t chunks = reach < 0 ? 0u : static_cast<std::uint32_t>(reach) / kChunkTokens + 1u;
    return (chunks + split_chunks - 1u) / split_chunks;
}

// Dims 4 d4 .. + 3 of a vector over splits of it: references, denominator and
// sums so far.
struct Joined {
    float ref = kNone;
    int lead = kNone2;
    float total = 0.0f;
    float4v acc = {0.f, 0.f, 0.f, 0.f};
};

__device__ __forceinline__ void join(Joined& x, float ref, int lead, float total, const float4v& acc) {
    const float next = ref > x.ref ? ref : x.ref;
    const int mine_down = powers(x.ref - next), down = powers(ref - next);
    const int mine = x.lead + mine_down > kNone2 ? x.lead + mine_down : kNone2, theirs = lead + down;
    const int next_lead = theirs > mine ? theirs : mine;
    x.total = __builtin_amdgcn_ldexpf(x.total, mine_down) + __builtin_amdgcn_ldexpf(total, down);
#pragma unroll
    for (unsigned r = 0; r < 4u; ++r) {
        x.acc[r] = __builtin_amdgcn_ldexpf(x.acc[r], mine - next_lead) + __builtin_amdgcn_ldexpf(acc[r], theirs - next_lead);
    }
    x.ref = next;
    x.lead = next_lead;
}

// Splits begin .. end - 1 of a vector's partials, eight loads in flight.
template <unsigned D>
__device__ __forceinline__ Joined join_splits(const float* __restrict__ base, std::uint32_t begin, std::uint32_t end,
                                              unsigned d4) {
    constexpr unsigned kBatch = 8;
    Joined x;
    for (std::uint32_t s0 = begin; s0 < end; s0 += kBatch) {
        float4v head[kBatch], sums[kBatch];
#pragma unroll
        for (unsigned j = 0; j < kBatch; ++j) {
            const std::uint32_t at = (s0 + j < end ? s0 + j : end - 1u) * (D + kStat);
            head[j] = *reinterpret_cast<const float4v*>(base + at);
            sums[j] = *reinterpret_cast<const float4v*>(base + at + kStat + 4u * d4);
        }
#pragma unroll
        for (unsigned j = 0; j < kBatch; ++j) {
            if (s0 + j < end) join(x, head[j][0], __float_as_int(head[j][1]), head[j][2], sums[j]);
        }
    }
    return x;
}

__device__ __forceinline__ float4v normalised(const Joined& x) {
    float4v y;
#pragma unroll
    for (unsigned r = 0; r < 4u; ++r) {
        y[r] = x.total == 0.0f ? 0.0f : __builtin_amdgcn_ldexpf(x.acc[r] / x.total, x.lead - kPBits);
    }
    return y;
}

// Joins the splits of a tile's vectors.  A launch of its own costs 4 us here;
// what it reads (a few MB) costs less.  WIDE, for more than 16 splits: a
// workgroup a vector, whose threads take a slice of the splits each and meet
// in LDS (one row of 2 x 7 heads over 131072 tokens, 256 splits: 24 us with the
// attention, 70 where a thread joins all of them).
template <unsigned D, unsigned NV, bool RUNS, bool WIDE>
__global__ __launch_bounds__(kThreads) void kv8_merge_kernel(
    const std::int32_t* __restrict__ positions, std::uint32_t m, std::uint32_t q_heads, std::uint32_t kv_heads,
    const std::int32_t* __restrict__ run_starts, std::uint32_t runs, std::uint32_t tile_rows, std::uint64_t max_tokens,
    Kv8Cut cut, const float* __restrict__ partials, float2* __restrict__ stats, float* __restrict__ out) {
    constexpr unsigned kTile = kVectors * NV;
    constexpr unsigned kPieces = D / 4u, kSlices = WIDE ? kThreads / kPieces : 1u;
    const std::uint32_t group = q_heads / kv_heads, parts = (group + kTile - 1u) / kTile;
    const Kv8Work work = kv8_work(cut, cut.whole + blockIdx.x, kv_heads * parts);
    const std::uint32_t kvh = work.tile_head / parts, part = work.tile_head % parts;
    Tile tile{work.tile, 1u, 0u, 0u};
    if constexpr (RUNS) tile = find_tile(work.tile, cut.pairs / (kv_heads * parts), run_starts, runs, m, tile_rows);
    if (tile.rows == 0u) return;
    tile.head = kvh * group + part * kTile;
    tile.heads = group - part * kTile < kTile ? group - part * kTile : kTile;
    int reach = -1;
    for (unsigned r = 0; r < tile.rows; ++r) {
        const int p = positions[tile.row + r];
        reach = p > reach ? p : reach;
    }
    const std::uint32_t live = live_splits(reach, max_tokens, cut.split_chunks), splits = cut.splits;
    if (live <= 1u) return;   // the attention kernel wrote this tile
    const unsigned d4 = threadIdx.x % kPieces, slice = WIDE ? threadIdx.x / kPieces : 0u;
    const unsigned step = WIDE ? 1u : kThreads / kPieces;   // vectors at a time
    for (unsigned v = blockIdx.y * step + (WIDE ? 0u : threadIdx.x / kPieces); v < tile.rows * tile.heads;
         v += gridDim.y * step) {
        const std::uint64_t vector =
            static_cast<std::uint64_t>(tile.row + v / tile.heads) * q_heads + tile.head + v % tile.heads;
        const std::uint64_t place = RUNS ? static_cast<std::uint64_t>(blockIdx.x) * kTile + v : vector;
        const float* const base = partials + place * splits * (D + kStat);
        const std::uint32_t each = (live + kSlices - 1u) / kSlices, from = slice * each < live ? slice * each : live;
        Joined x = join_splits<D>(base, from, live - from < each ? live : from + each, d4);
        if constexpr (WIDE) {
            __shared__ float4v sums[kSlices][kPieces];
            __shared__ float refs[kSlices], totals[kSlices];
            __shared__ int leads[kSlices];
            __syncthreads();   // the vector before is out
            sums[slice][d4] = x.acc;
            if (d4 == 0u) {
                refs[slice] = x.ref;
                leads[slice] = x.lead;
                totals[slice] = x.total;
            }
            __syncthreads();
            if (slice != 0u) continue;
#pragma unroll
            for (unsigned w = 1; w < kSlices; ++w) join(x, refs[w], leads[w], totals[w], sums[w][d4]);
        }
        *reinterpret_cast<float4v*>(out + vector * D + 4u * d4) = normalised(x);
        if (stats && d4 == 0u) {
            stats[vector] = make_float2(x.ref, x.total == 0.0f ? 0.0f : 1.0f / x.total);
        }
    }
}

// A step of the sum over 16 vectors: lanes W apart exchange halves of what
// they hold, so after steps 8, 4, 2 and 1 lane col has token col's sum.
template <unsigned W>
__device__ __forceinline__ void halve(float (&sum)[16], unsigned col) {
    const bool upper = (col & W) != 0u;
#pragma unroll
    for (unsigned t = 0; t < W; ++t) {
        const float keep = upper ? sum[t + W] : sum[t], give = upper ? sum[t] : sum[t + W];
        sum[t] = keep + __shfl_xor(give, W);
    }
}

// The last position of rows begin..end - 1, at most `most`, in every lane.
__device__ __forceinline__ int last_position(const std::int32_t* __restrict__ positions, std::int64_t begin,
                                             std::int64_t end, unsigned lane, int most) {
    int last = -1;
    for (std::int64_t r = begin + lane; r < end; r += 64) last = positions[r] > last ? positions[r] : last;
    for (int off = 32; off > 0; off >>= 1) {
        const int o = __shfl_xor(last, off);
        last = o > last ? o : last;
    }
    return last < most ? last : most;
}

// A token's weight to its record, if the token is held.
__device__ __forceinline__ void put_weight(Kv8Byte* record, int first, int last, unsigned col, float weight, bool add) {
    if (record == nullptr || first + static_cast<int>(col) > last) return;
    float* const at = (float*)(record + kKv8Weights) + col;
    if (add) {
        atomicAdd(at, weight);
    } else {
        *at = weight;
    }
}

// A chunk's records: each lane looks one of the four blocks up (so two loads
// follow on each other, not four), of which `page` is the page, and the wave
// shares them.
struct ChunkRecords {
    Kv8Byte* key;      // of the block whose K this lane loads
    Kv8Byte* value;    // of block lane / 16
};

__device__ __forceinline__ ChunkRecords chunk_records(const Kv8Geometry& g, std::int32_t page, std::uint32_t slot,
                                                      std::uint32_t layer, std::uint32_t kvh, std::uint32_t chunk,
                                                      unsigned lane) {
    Kv8Byte* const mine = kv8_record_in(g, page, slot, layer, kvh, chunk * kChunkBlocks + (lane & 3u));
    const std::uint64_t address = reinterpret_cast<std::uint64_t>((unsigned char*)mine);
    const int low = static_cast<int>(address), high = static_cast<int>(address >> 32);
    const auto of = [&](unsigned b) __attribute__((always_inline)) {
        const std::uint64_t h = static_cast<std::uint32_t>(__shfl(high, b));
        return (Kv8Byte*)(h << 32 | static_cast<std::uint32_t>(__shfl(low, b)));
    };
    return ChunkRecords{of((lane & 15u) >> 2), of(lane >> 4)};
}

// The weights a run's rows give one chunk of tokens: the scores again, by the
// same instructions as in the attention, and p from the rows' statistics
// (M and 1 / l).  Reading K again takes half of the attention's bytes; keeping
// the scores would take 4 bytes a vector and token, written and read.  Each
// token takes one atomic addition: a page that two runs share loses nothing,
// and elsewhere a single addition leaves one order.
//
// A chunk of a (run, KV head) is one wave's, which takes the run's vectors 16
// at a time.  MERGE, where single rows were split up to 16 times: the grid's
// first column joins the splits of a run's rows, and the others take the
// statistics from the partials themselves, so that one launch follows the
// attention.
template <int TYPE, unsigned D, bool MERGE>
__global__ __launch_bounds__(kThreads, 3) void kv8_weights_kernel(
    Kv8Geometry g, const float* __restrict__ qkv, std::uint64_t stride, std::uint32_t m,
    const std::int32_t* __restrict__ positions, const std::int32_t* __restrict__ tables, std::uint32_t layer,
    std::uint32_t q_heads, const std::int32_t* __restrict__ run_starts, std::uint64_t max_tokens, float score_scale,
    const float2* __restrict__ stats, bool add, std::uint32_t split_chunks, std::uint32_t splits,
    const float* __restrict__ partials, float* __restrict__ out) {
    const unsigned tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, grp = lane >> 4, col = lane & 15u;
    const std::uint32_t kvh = blockIdx.y, run = blockIdx.z;
    std::int64_t begin = run, end = static_cast<std::int64_t>(run) + 1;
    if (run_starts) {
        begin = run_starts[run];
        end = run_starts[run + 1u];
    }
    begin = begin < 0 ? 0 : begin;
    end = end > static_cast<std::int64_t>(m) ? static_cast<std::int64_t>(m) : end;
    if (begin >= end) return;
    const std::uint32_t group = q_heads / g.kv_heads;
    const std::uint32_t vectors = static_cast<std::uint32_t>(end - begin) * group;
    const std::uint32_t row0 = static_cast<std::uint32_t>(begin), head0 = kvh * group;
    if (MERGE && blockIdx.x == 0u) {
        for (unsigned idx = tid; idx < vectors * (D / 4u); idx += kThreads) {
            const unsigned v = idx / (D / 4u), d4 = idx % (D / 4u);
            const std::uint32_t r = row0 + v / group;
            const std::uint64_t vector = static_cast<std::uint64_t>(r) * q_heads + head0 + v % group;
            const std::uint32_t live = live_splits(positions[r], max_tokens, split_chunks);
            if (live <= 1u) continue;   // the attention kernel wrote this row
            *reinterpret_cast<float4v*>(out + vector * D + 4u * d4) =
                normalised(join_splits<D>(partials + vector * splits * (D + kStat), 0u, live, d4));
        }
        return;
    }
    const std::uint32_t column = blockIdx.x - (MERGE ? 1u : 0u);
    const std::uint32_t chunk = column * kWaves + wave;
    const int token0 = static_cast<int>(chunk * kChunkTokens);
    const std::int32_t* const table = tables + static_cast<std::uint64_t>(row0) * g.max_pages;
    const std::uint32_t slot = kv8_slot(g, chunk * kChunkBlocks + (lane & 3u));
    const std::int32_t page = slot < g.max_pages ? table[slot] : -1;
    // Tokens past the run's last position (or max_tokens) are not held.
    const int most = static_cast<int>(max_tokens) - 1;
    const int last = last_position(positions, begin, end, lane, most);
    if (token0 > last) return;
    const Kv8Byte* const none = (const Kv8Byte*)g_no_record;
    const ChunkRecords at = chunk_records(g, page, slot, layer, kvh, chunk, lane);
    const Kv8Byte* const krec = at.key;
    Kv8Byte* const vrec = at.value;
    KeyCodes<D> keys;
    load_keys<D>(krec ? krec : none, lane, keys);
    const float k_scale = load_scales(vrec ? vrec : none).x;
    const int first = token0 + static_cast<int>(grp * kKv8Block);
    float sum[16] = {};
    for (std::uint32_t v0 = 0u; v0 < vectors; v0 += kVectors) {
        const std::uint32_t v = v0 + col;
        const bool active = v < vectors;
        const std::uint32_t r = row0 + (active ? v / group : 0u);
        const std::uint64_t vector = static_cast<std::uint64_t>(r) * q_heads + head0 + (active ? v % group : 0u);
        const int position = positions[r];
        int upto = active ? position : -1;
        upto = upto < most ? upto : most;
        if (!__any(upto >= token0)) continue;
        QueryFragments<D> q;
        load_query<D>(active ? qkv + static_cast<std::uint64_t>(r) * stride + (vector - static_cast<std::uint64_t>(r) * q_heads) * D
                             : nullptr,
                      grp, q);
        float base, share;   // M and 1 / l
        const std::uint32_t live = MERGE ? live_splits(position, max_tokens, split_chunks) : 1u;
        if (MERGE && __any(live > 1u)) {
            // Lane group grp takes splits grp, grp + 4, ...; then they meet.
            float ref = kNone, total = 0.0f;
            for (std::uint32_t s = grp; s < live && live > 1u; s += 4u) {
                const float4v head = *reinterpret_cast<const float4v*>(partials + (vector * splits + s) * (D + kStat));
                const float next = head[0] > ref ? head[0] : ref;
                total = __builtin_amdgcn_ldexpf(total, powers(ref - next)) + __builtin_amdgcn_ldexpf(head[2], powers(head[0] - next));
                ref = next;
            }
            base = groups_max(ref);
            total = __builtin_amdgcn_ldexpf(total, powers(ref - base));
            total += __shfl_xor(total, 16);
            total += __shfl_xor(total, 32);
            share = total == 0.0f ? 0.0f : 1.0f / total;
            if (live <= 1u) {   // the attention kernel left this row's
                const float2 st = stats[vector];
                base = st.x;
                share = st.y;
            }
        } else {
            const float2 st = stats[vector];
            base = st.x;
            share = st.y;
        }
        float4v s[4];
        chunk_scores<TYPE, D>(keys, q, s);
        float factor = score_factor(q.undo * score_scale, k_scale);
        round_large<TYPE, D>(s, factor);
        const int limit = vrec == nullptr ? -1 : upto - first;
#pragma unroll
        for (unsigned t = 0; t < 16u; ++t) {
            const float p = score_power(s[t >> 2][t & 3u], factor, base) * share;
            sum[t] += static_cast<int>(t) <= limit ? p : 0.0f;
        }
    }
    halve<8>(sum, col);
    halve<4>(sum, col);
    halve<2>(sum, col);
    halve<1>(sum, col);
    put_weight(vrec, first, last, col, sum[0], add);
}

// The same for runs of many vectors: a chunk is a workgroup's, whose waves take
// the vectors 16 at a time in turn and add up in LDS.  The attention left the
// vectors' operands, and a wave reads 16 vectors ahead (four runs of 32 rows
// over 2900..4100 tokens, 28 q heads on 4 KV heads of 128 dims: 30 us where
// every chunk made the operands anew, 25 reading them, 22.7 reading ahead and
// with K's codes as f16 in registers for all vectors).
template <int TYPE, unsigned D>
__global__ __launch_bounds__(kThreads, 2) void kv8_run_weights_kernel(
    Kv8Geometry g, std::uint32_t m, const std::int32_t* __restrict__ positions, const std::int32_t* __restrict__ tables,
    std::uint32_t layer, std::uint32_t q_heads, const std::int32_t* __restrict__ run_starts, std::uint64_t max_tokens,
    float score_scale, const float2* __restrict__ stats, const half8v* __restrict__ queries,
    const float* __restrict__ undos, bool add) {
    __shared__ float shared_sum[kWaves][kChunkTokens];
    const unsigned tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, grp = lane >> 4, col = lane & 15u;
    const std::uint32_t kvh = blockIdx.y, run = blockIdx.z, chunk = blockIdx.x;
    std::int64_t begin = run_starts[run], end = run_starts[run + 1u];
    begin = begin < 0 ? 0 : begin;
    end = end > static_cast<std::int64_t>(m) ? static_cast<std::int64_t>(m) : end;
    if (begin >= end) return;
    const std::uint32_t group = q_heads / g.kv_heads;
    const std::uint32_t vectors = static_cast<std::uint32_t>(end - begin) * group;
    const std::uint32_t row0 = static_cast<std::uint32_t>(begin), head0 = kvh * group;
    const std::int32_t* const table = tables + static_cast<std::uint64_t>(row0) * g.max_pages;
    const std::uint32_t slot = kv8_slot(g, chunk * kChunkBlocks + (lane & 3u));
    const std::int32_t page = slot < g.max_pages ? table[slot] : -1;
    // Tokens past the run's last position (or max_tokens) are not held.
    const int most = static_cast<int>(max_tokens) - 1;
    const int last = last_position(positions, begin, end, lane, most);
    const int token0 = static_cast<int>(chunk * kChunkTokens);
    if (token0 > last) return;   // all of the workgroup's waves
    const ChunkRecords at = chunk_records(g, page, slot, layer, kvh, chunk, lane);
    const Kv8Byte* const none = (const Kv8Byte*)g_no_record;
    half8v a[4][D / 32];
    {
        KeyCodes<D> keys;
        load_keys<D>(at.key ? (const Kv8Byte*)at.key : none, lane, keys);
#pragma unroll
        for (unsigned b = 0; b < 4u; ++b) {
#pragma unroll
            for (unsigned i = 0; i < D / 64u; ++i) codes_to_half<TYPE>(keys.c[b][i], a[b][2u * i], a[b][2u * i + 1u]);
        }
    }
    const float k_scale = load_scales(at.value ? (const Kv8Byte*)at.value : none).x;
    const int first = token0 + static_cast<int>(grp * kKv8Block);
    float sum[16] = {};
    struct Vector {
        QueryFragments<D> q;
        float2 st;
        int upto;
    };
    const auto fetch = [&](std::uint32_t v0, Vector& x) __attribute__((always_inline)) {
        const bool active = v0 + col < vectors;   // places without a vector repeat the first
        const std::uint32_t v = active ? v0 + col : 0u, r = row0 + v / group;
        const std::uint64_t vector = static_cast<std::uint64_t>(r) * q_heads + head0 + v % group;
        x.upto = positions[r];
        x.st = stats[vector];
        x.q.undo = undos[vector];
        kept_query<D>(queries + vector * (D / 4u), grp, x.q);
    };
    Vector now;
    fetch(wave * kVectors, now);
    for (std::uint32_t v0 = wave * kVectors; v0 < vectors; v0 += kWaves * kVectors) {
        Vector next;
        fetch(v0 + kWaves * kVectors, next);
        const int upto = v0 + col < vectors ? (now.upto < most ? now.upto : most) : -1;
        const int limit = at.value == nullptr ? -1 : upto - first;
        if (__any(limit >= 0)) {
            float4v s[4];
#pragma unroll
            for (unsigned b = 0; b < 4u; ++b) {
                s[b] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (unsigned i = 0; i < D / 16u; ++i) {   // low parts first
                    s[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[b][i % (D / 32u)], i < D / 32u ? now.q.lo[i] : now.q.hi[i - D / 32u],
                                                                  s[b], 0, 0, 0);
                }
            }
            float factor = score_factor(now.q.undo * score_scale, k_scale);
            round_large<TYPE, D>(s, factor);
            if (__all(limit >= 15)) {
#pragma unroll
                for (unsigned t = 0; t < 16u; ++t) {
                    sum[t] = __builtin_fmaf(score_power(s[t >> 2][t & 3u], factor, now.st.x), now.st.y, sum[t]);
                }
            } else {
#pragma unroll
                for (unsigned t = 0; t < 16u; ++t) {
                    const float p = score_power(s[t >> 2][t & 3u], factor, now.st.x);
                    sum[t] = static_cast<int>(t) <= limit ? __builtin_fmaf(p, now.st.y, sum[t]) : sum[t];
                }
            }
        }
        now = next;
    }
    halve<8>(sum, col);
    halve<4>(sum, col);
    halve<2>(sum, col);
    halve<1>(sum, col);
    shared_sum[wave][lane] = sum[0];
    __syncthreads();
    if (wave != 0u) return;
    float mine = 0.0f;
#pragma unroll
    for (unsigned w = 0; w < kWaves; ++w) mine += shared_sum[w][lane];
    put_weight(at.value, first, last, col, mine, add);
}

} // namespace

Kv8Shape kv8_attention_shape(std::uint32_t m, std::uint32_t q_heads, std::uint32_t kv_heads, std::uint32_t head_dim,
                             std::uint32_t runs, std::uint64_t max_tokens, bool weights) {
    const std::uint32_t group = q_heads / kv_heads;
    const std::uint32_t chunks = static_cast<std::uint32_t>((max_tokens + kChunkTokens - 1u) / kChunkTokens);
    const std::uint32_t row_parts = (group + kVectors - 1u) / kVectors;
    const std::uint64_t row_pairs = static_cast<std::uint64_t>(m) * kv_heads * row_parts;
    // Tiles of runs, as if all runs were of one length: a chunk of one costs
    // as much as that of 1.6 single rows, and about 5 us more a call.  Over
    // 660 calls (1..24 runs of 2..512 rows over up to 3000 tokens, 8 x 1, 8 x
    // 2, 8 x 4, 4 x 7, 2 x 14 and 8 x 16 heads of 64 and 128 dims) this takes
    // 0.7 % longer in the mean than the better of both, 30 % at most; runs'
    // tiles always took 18 % longer, up to 1.8 times.  Runs of one call were
    // of about one length there.  63 rows of a decode step and a prompt's 512 in
    // one call, 4 x 7 heads over 4000 tokens, take 136 us (43 and 79 in calls of
    // their own), with weights 565 (78 and 136).
    const std::uint32_t run_rows = runs != 0u ? (m + runs - 1u) / runs : 0u;
    const std::uint32_t tile = kVectors * kRunTiles, parts = (group + tile - 1u) / tile;
    const std::uint32_t tile_rows = group < tile ? tile / group : 1u;
    const std::uint64_t run_pairs = static_cast<std::uint64_t>(runs) * ((run_rows + tile_rows - 1u) / tile_rows) * kv_heads * parts;
    const bool by_work = 5u * row_pairs * (chunks + 2u) > 8u * run_pairs * (chunks + 2u) + 20000u;
    // A run's weights: a wave a chunk takes its vectors one 16 after the other,
    // which suits chunks for all SIMDs (24 runs of 24 rows over 3000 tokens, 8
    // heads: 76 us against 105), and a workgroup a chunk does many vectors with
    // few chunks (4 runs of 100 rows from the start: 26 against 19).  The second
    // needs the vectors that runs' tiles leave, and is worth them from 80 on
    // (a prompt of 512 rows, 4 x 7 heads: 397 us without, 65).
    const std::uint64_t run_vectors = static_cast<std::uint64_t>(run_rows) * group;
    const bool run_weights =
        weights && 400u * ((run_vectors + kVectors - 1u) / kVectors) > static_cast<std::uint64_t>(runs) * kv_heads * chunks;
    if (runs != 0u && (by_work || (weights && run_vectors >= 80u))) {
        const std::uint64_t pairs = (static_cast<std::uint64_t>(m / tile_rows) + runs) * kv_heads * parts;
        // Workgroups that run at a time: two a CU, with the registers of two
        // MFMA tiles of 128 dims, or three.  What fills them is not cut; the
        // pairs left over are, so that they fill them once more together (of
        // them about as many hold a tile as if all runs were of one length).
        const std::uint64_t slots = head_dim == 128u ? 512u : 768u;
        const std::uint64_t whole = chunks >= 4u * kWaves ? pairs / slots * slots : pairs;
        std::uint64_t per = chunks;
        if (pairs > whole) {
            const std::uint64_t left = (pairs - whole) * (run_pairs < pairs ? run_pairs : pairs) / pairs;
            const std::uint64_t splits = slots / (left > 0u ? left : 1u);
            per = (chunks + splits - 1u) / splits;
            per = (per + kWaves - 1u) / kWaves * kWaves;
            if (per < 2u * kWaves) per = 2u * kWaves;
            if (per > chunks) per = chunks;
        }
        const std::uint32_t splits = static_cast<std::uint32_t>((chunks + per - 1u) / per);
        return Kv8Shape{{static_cast<std::uint32_t>(pairs), static_cast<std::uint32_t>(splits > 1u ? whole : 0u), splits,
                         static_cast<std::uint32_t>(per)},
                        tile_rows, kKv8Runs, run_weights};
    }
    const auto shape = [&](std::uint64_t per, int kernel) {
        return Kv8Shape{{static_cast<std::uint32_t>(row_pairs), 0u, static_cast<std::uint32_t>((chunks + per - 1u) / per),
                         static_cast<std::uint32_t>(per)},
                        0u, kernel, false};
    };
    // Single rows, by the best of seven ways over 510 calls of equal and 510 of
    // unequal lengths (1..128 rows, up to 16000 tokens, lengths within a factor of
    // four, 2 x 7, 4 x 7 and 8 x 4 heads): this rule lies 2.4 and 0.8 % off it in
    // the mean and 20 % at most.
    //
    // Eight waves a workgroup and one launch: up to two turns of the waves (32
    // rows of 4 x 7 heads over 500..1200 tokens 11.5 us, 14.2 in splits), four
    // with workgroups for half of the CUs, and any number where they fill
    // them (64 such rows over 3000 tokens 34 us, 38 in splits; 40 over 60000
    // 478, 516 in splits).  That is for lengths much alike: of 40 rows one over
    // 131072 tokens and the others over 1000, the long one's four workgroups walk
    // 747 us, where splits take 278 (one over 16000: 97, 47).
    const bool full = head_dim == 128u && row_pairs >= 160u;
    if (row_pairs <= 256u && (chunks <= 16u || (chunks <= 32u && row_pairs >= 128u) || full)) {
        return shape(chunks, kKv8ShortRows);
    }
    // More short rows than that: the splits' meeting would cost more than they
    // even out (128 rows over 600 tokens 19 us, 25 in splits).
    if (chunks <= 48u && row_pairs >= 320u) return shape(chunks, kKv8Rows);
    // Splits of equal length, so that rows of unequal lengths make workgroups
    // of equal work, as many as run at a time if every row were max_tokens
    // long: three a CU, or four with the registers of 64 dims.  At least a
    // chunk a wave (one row over 2000 tokens 11 us, 19 unsplit), two where
    // there are many.
    const std::uint64_t slots = head_dim == 128u ? 768u : 1024u, least = chunks <= 32u ? kWaves : 2u * kWaves;
    std::uint64_t per = (row_pairs * chunks + slots - 1u) / slots;
    per = (per + kWaves - 1u) / kWaves * kWaves;
    if (per < least) per = least;
    return shape(per > chunks ? chunks : per, kKv8Rows);
}

namespace {

// The parts of the scratch memory: rows' statistics, and for runs of several
// rows their vectors' operands, where weights are gathered; splits' partials.
struct Scratch {
    std::uint64_t queries, undos, partials, bytes;
};

// places: vectors' splits.
Scratch scratch_parts(std::uint64_t vectors, std::uint32_t head_dim, bool weights, bool keep, std::uint64_t places) {
    const auto padded = [](std::uint64_t bytes) { return (bytes + 255u) / 256u * 256u; };
    Scratch s{};
    s.queries = weights ? padded(vectors * sizeof(float2)) : 0u;
    s.undos = s.queries + (keep ? vectors * head_dim * 2u * sizeof(_Float16) : 0u);
    s.partials = s.undos + (keep ? padded(vectors * sizeof(float)) : 0u);
    s.bytes = s.partials + places * (head_dim + kStat) * sizeof(float);
    return s;
}

Scratch scratch_of(const Kv8Shape& shape, std::uint32_t m, std::uint32_t q_heads, std::uint32_t head_dim, bool weights) {
    const std::uint64_t vectors = static_cast<std::uint64_t>(m) * q_heads;
    // Of runs the tiles that are cut have a place a vector, of rows all vectors.
    const std::uint64_t cut = shape.kernel == kKv8Runs
                                  ? static_cast<std::uint64_t>(shape.cut.pairs - shape.cut.whole) * kVectors * kRunTiles
                                  : vectors;
    return scratch_parts(vectors, head_dim, weights, shape.run_weights, shape.cut.splits > 1u ? cut * shape.cut.splits : 0u);
}

} // namespace

// What a call asks for is not what its shape takes, which falls where more rows
// need fewer splits, but a bound that grows with m, runs, max_tokens and
// weights: a call with the largest of each leaves room for all others, so that
// none of them allocates while it is captured.
//
// Splits of single rows hold at least kWaves chunks, and there is more than one
// only of less pairs than slots, when pairs * splits < slots + pairs.  Tiles are
// cut from 4 kWaves chunks on, less of them than slots, into splits of at least
// 2 kWaves chunks; run_pairs is at least half of pairs, so with the rounding
// of `left` tiles * splits is at most 3 slots.
std::uint64_t kv8_attention_scratch(std::uint32_t m, std::uint32_t q_heads, std::uint32_t kv_heads, std::uint32_t head_dim,
                                    std::uint32_t runs, std::uint64_t max_tokens, bool weights) {
    const auto least = [](std::uint64_t a, std::uint64_t b) { return a < b ? a : b; };
    const std::uint64_t chunks = (max_tokens + kChunkTokens - 1u) / kChunkTokens, group = q_heads / kv_heads;
    const std::uint64_t row_parts = (group + kVectors - 1u) / kVectors, row_slots = head_dim == 128u ? 768u : 1024u;
    const std::uint64_t row_splits = least(m * kv_heads * row_parts * ((chunks + kWaves - 1u) / kWaves), 2u * row_slots);
    std::uint64_t places = chunks > kWaves ? row_splits * ((group + row_parts - 1u) / row_parts) : 0u;
    if (runs != 0u && chunks >= 4u * kWaves) {
        const std::uint64_t tile = kVectors * kRunTiles, parts = (group + tile - 1u) / tile;
        const std::uint64_t tiles = (m / (group < tile ? tile / group : 1u) + runs) * kv_heads * parts;
        const std::uint64_t slots = head_dim == 128u ? 512u : 768u;
        const std::uint64_t splits = least(least(tiles, slots) * ((chunks + 2u * kWaves - 1u) / (2u * kWaves)), 3u * slots);
        places = places > splits * tile ? places : splits * tile;
    }
    return scratch_parts(static_cast<std::uint64_t>(m) * q_heads, head_dim, weights, weights && runs != 0u, places).bytes;
}

namespace {

template <int TYPE, unsigned D>
void launch_typed(const Kv8Geometry& g, const float* qkv, std::uint64_t stride, std::uint32_t m,
                  const std::int32_t* positions, const std::int32_t* tables, std::uint32_t layer, std::uint32_t q_heads,
                  const std::int32_t* run_starts, std::uint32_t runs, std::uint64_t max_tokens, int weights,
                  const Kv8Shape& shape, float* partials, float2* stats, half8v* queries, float* undos, float* out,
                  hipStream_t stream) {
    // Scores in powers of two: s log2(e) = (q . k) * log2(e) / sqrt(D).
    const float scale = static_cast<float>(1.4426950408889634 / __builtin_sqrt(static_cast<double>(D)));
    const Kv8Cut& cut = shape.cut;
    const bool split = cut.splits > 1u, by_run = shape.kernel == kKv8Runs;
    const dim3 grid(cut.whole + (cut.pairs - cut.whole) * cut.splits);
    // A tile of several MFMA tiles is joined by several workgroups, and one of
    // many splits by one a vector.
    const bool wide = cut.splits > 16u;
    const dim3 merge_grid(cut.pairs - cut.whole, wide ? kVectors : by_run ? 4u : 1u);
#define AIR_KV8_ATTENTION(NV, RUNS, W)                                                                               \
    hipLaunchKernelGGL((kv8_attention_kernel<TYPE, D, NV, RUNS, W>), grid, dim3(64 * W), 0, stream, g, qkv, stride, m, \
                       positions, tables, layer, q_heads, run_starts, runs, shape.tile_rows, max_tokens, cut, scale, \
                       partials, stats, queries, undos, out)
#define AIR_KV8_MERGE_KERNEL(NV, RUNS, WIDE)                                                                         \
    hipLaunchKernelGGL((kv8_merge_kernel<D, NV, RUNS, WIDE>), merge_grid, dim3(kThreads), 0, stream, positions, m, q_heads, \
                       g.kv_heads, run_starts, runs, shape.tile_rows, max_tokens, cut, partials, stats, out)
#define AIR_KV8_MERGE(NV, RUNS)                         \
    do {                                                \
        if (wide) AIR_KV8_MERGE_KERNEL(NV, RUNS, true); \
        else AIR_KV8_MERGE_KERNEL(NV, RUNS, false);     \
    } while (false)
#define AIR_KV8_WEIGHTS(MERGE, COLUMNS)                                                                              \
    hipLaunchKernelGGL((kv8_weights_kernel<TYPE, D, MERGE>), dim3(COLUMNS, g.kv_heads, run_starts ? runs : m), \
                       dim3(kThreads), 0, stream, g, qkv, stride, m, positions, tables, layer, q_heads, run_starts,  \
                       max_tokens, scale, stats, weights == 1, cut.split_chunks, cut.splits, partials, out)
    const std::uint32_t chunks = static_cast<std::uint32_t>((max_tokens + kChunkTokens - 1u) / kChunkTokens);
    const std::uint32_t columns = (chunks + kWaves - 1u) / kWaves;
    if (by_run) {
        AIR_KV8_ATTENTION(kRunTiles, true, kWaves);
        if (split) AIR_KV8_MERGE(kRunTiles, true);
        if (weights && !shape.run_weights) AIR_KV8_WEIGHTS(false, columns);
        if (shape.run_weights) {
            hipLaunchKernelGGL((kv8_run_weights_kernel<TYPE, D>), dim3(chunks, g.kv_heads, runs), dim3(kThreads), 0, stream, g,
                               m, positions, tables, layer, q_heads, run_starts, max_tokens, scale, stats, queries, undos,
                               weights == 1);
        }
    } else {
        if (shape.kernel == kKv8ShortRows) AIR_KV8_ATTENTION(1u, false, kShortWaves);
        else AIR_KV8_ATTENTION(1u, false, kWaves);
        const bool together = weights && split && !wide;   // splits and weights in one launch
        if (together) AIR_KV8_WEIGHTS(true, columns + 1u);
        if (split && !together) AIR_KV8_MERGE(1u, false);
        if (weights && !together) AIR_KV8_WEIGHTS(false, columns);
    }
#undef AIR_KV8_ATTENTION
#undef AIR_KV8_MERGE
#undef AIR_KV8_MERGE_KERNEL
#undef AIR_KV8_WEIGHTS
}

} // namespace

hipError_t launch_kv8_attention(const Kv8Geometry& g, const float* qkv, std::uint64_t stride, std::uint32_t m,
                                const std::int32_t* positions, const std::int32_t* tables, std::uint32_t layer,
                                std::uint32_t q_heads, const std::int32_t* run_starts, std::uint32_t runs,
                                std::uint64_t max_tokens, int weights, const Kv8Shape& shape, void* scratch, float* out,
                                hipStream_t stream) {
    const Scratch at = scratch_of(shape, m, q_heads, g.head_dim, weights != 0);
    unsigned char* const base = static_cast<unsigned char*>(scratch);
    float2* const stats = weights ? reinterpret_cast<float2*>(base) : nullptr;
    const bool keep = shape.run_weights;
    half8v* const queries = keep ? reinterpret_cast<half8v*>(base + at.queries) : nullptr;
    float* const undos = keep ? reinterpret_cast<float*>(base + at.undos) : nullptr;
    float* const partials = reinterpret_cast<float*>(base + at.partials);
    const auto launch = g.type == kKv8I8 ? (g.head_dim == 128u ? launch_typed<kKv8I8, 128> : launch_typed<kKv8I8, 64>)
                                         : (g.head_dim == 128u ? launch_typed<kKv8E4M3, 128> : launch_typed<kKv8E4M3, 64>);
    launch(g, qkv, stride, m, positions, tables, layer, q_heads, run_starts, runs, max_tokens, weights, shape, partials,
           stats, queries, undos, out, stream);
    return hipGetLastError();
}

} // namespace air_hip

// rows.h -- rows of head_dim elements in fp32: eight consecutive elements per lane, so a row is
// head_dim / 8 lanes and a wave instruction covers 512 elements; what the attention operators share.
#pragma once

#include "vec.h"

namespace tccl {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef int16_t s16x2 __attribute__((ext_vector_type(2)));

struct PoolTable {
    char *p[TCCL_MAX_WORLD];
};

// Eight elements as they lie in memory, and in fp32.
struct Bf16Row {
    static constexpr int kElemBytes = 2;
    u32x4 raw;
    template <bool NT = false>
    __device__ __forceinline__ void load(const char *p)
    {
        raw = load_vec<NT>(p, 0);
    }
    __device__ __forceinline__ void zero() { raw = u32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ float at(int k) const
    {
        return bits_to_f32((k & 1) ? raw[k >> 1] & 0xFFFF0000u : raw[k >> 1] << 16);
    }
    // the largest magnitude's fp32 bits (integers in the order of the magnitudes; infinity and NaN above all)
    __device__ __forceinline__ uint32_t magnitude() const
    {
        u16x2 m = __builtin_bit_cast(u16x2, raw[0] & 0x7FFF7FFFu);
#pragma unroll
        for (int i = 1; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, raw[i] & 0x7FFF7FFFu));
        return static_cast<uint32_t>(m.x > m.y ? m.x : m.y) << 16;
    }
    // the eight elements divided by a power of two as e4m3 codes, rounded to nearest even; all finite
    __device__ __forceinline__ u32x2 codes(float scale) const
    {
        u32x2 r;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            s16x2 c = {0, 0};
            const uint32_t low = raw[2 * i], high = raw[2 * i + 1];
            c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, __builtin_bit_cast(bf16x2, low), scale, false);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, __builtin_bit_cast(bf16x2, high), scale, true);
            r[i] = __builtin_bit_cast(uint32_t, c);
        }
        return r;
    }
    static __device__ __forceinline__ void store(char *p, const float *x)
    {
        u32x4 r;
#pragma unroll
        for (int k = 0; k < 4; ++k) r[k] = pack_bf16(x[2 * k], x[2 * k + 1]);
        store_vec<false>(p, 0, r);
    }
};

struct F32Row {
    static constexpr int kElemBytes = 4;
    u32x4 raw[2];
    // never marked as streaming: the lane's two vectors share cache lines with its neighbours' (measured with one
    // source of 168 MB: 66 us plain, 75 streaming)
    template <bool NT = false>
    __device__ __forceinline__ void load(const char *p)
    {
        raw[0] = load_vec<false>(p, 0);
        raw[1] = load_vec<false>(p, 1);
    }
    __device__ __forceinline__ void zero() { raw[0] = raw[1] = u32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ float at(int k) const { return bits_to_f32(raw[k >> 2][k & 3]); }
    __device__ __forceinline__ uint32_t magnitude() const
    {
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t u = raw[k >> 2][k & 3] & 0x7FFFFFFFu;
            m = m > u ? m : u;
        }
        return m;
    }
    __device__ __forceinline__ u32x2 codes(float scale) const
    {
        u32x2 r;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            s16x2 c = {0, 0};
            c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, at(4 * i), at(4 * i + 1), scale, false);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, at(4 * i + 2), at(4 * i + 3), scale, true);
            r[i] = __builtin_bit_cast(uint32_t, c);
        }
        return r;
    }
    static __device__ __forceinline__ void store(char *p, const float *x)
    {
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            u32x4 r;
#pragma unroll
            for (int k = 0; k < 4; ++k) r[k] = f32_to_bits(x[4 * v + k]);
            store_vec<false>(p, v, r);
        }
    }
};

template <class Row>
__device__ __forceinline__ void load_row(const char *p, float *x)
{
    Row r;
    r.load(p);
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = r.at(k);
}

// x of another lane, by moves within rows of 16 lanes (no LDS round trip).
template <int CTRL>
__device__ __forceinline__ float dpp(float x)
{
    const int i = __builtin_bit_cast(int, x);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, CTRL, 0xF, 0xF, false));
}
constexpr int kDppXor1 = 0xB1, kDppXor2 = 0x4E, kDppHalfMirror = 0x141, kDppMirror = 0x140, kDppRotate8 = 0x128;

struct AddOp {
    static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
struct MaxOp {
    static __device__ __forceinline__ float of(float a, float b) { return fmaxf(a, b); }
};

// v_permlane16_swap of x with itself gives rows (0, 0, 2, 2) and (1, 1, 3, 3); v_permlane32_swap the
// lower and the upper half: their combination is the same in both partners.
template <class Op>
__device__ __forceinline__ float across16(float x)
{
    const uint32_t u = f32_to_bits(x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return Op::of(bits_to_f32(r[0]), bits_to_f32(r[1]));
}
template <class Op>
__device__ __forceinline__ float across32(float x)
{
    const uint32_t u = f32_to_bits(x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return Op::of(bits_to_f32(r[0]), bits_to_f32(r[1]));
}

// Over the LANES = 8, 16 or 32 neighbouring lanes of a row; every lane gets the result.
template <class Op, int LANES>
__device__ __forceinline__ float reduce_row(float x)
{
    static_assert(LANES == 8 || LANES == 16 || LANES == 32);
    x = Op::of(x, dpp<kDppXor1>(x));
    x = Op::of(x, dpp<kDppXor2>(x));
    x = Op::of(x, dpp<kDppHalfMirror>(x));
    if constexpr (LANES >= 16) x = Op::of(x, dpp<kDppMirror>(x));
    if constexpr (LANES == 32) x = across16<Op>(x);
    return x;
}

// ------------------------------------------------------------------ the paged cache's layout
// One rank's buffer is [pages_per_rank][kv_heads] blocks; a block holds one head of one page:
//   K        tiles of 16 tokens, each [head_dim / kChunk][16 tokens, see key_row][kChunk elements]; a chunk is 16 bytes
//   V        groups of kChunk tokens, each [head_dim][kChunk tokens]; again 16 bytes per dim
//   K and V exponents, one byte (exponent + 127) per token each (8-bit storage only)
// A wave's 16-byte loads of it are the operands of the attention's matrix instructions as they stand:
// keys with their dims along the contraction, values with their tokens along it.
struct Bf16Store {
    static constexpr int kBytes = 2;
    static constexpr int kChunk = 8; // elements in 16 bytes: dims of a K chunk, tokens of a V group
    static constexpr bool kScaled = false;
};
struct E4m3Store {
    static constexpr int kBytes = 1;
    static constexpr int kChunk = 16;
    static constexpr bool kScaled = true;
};

// A token's row in its K tile.  An attention load takes four tokens of each of two 8-token groups (bf16): they lie side
// by side, a whole 128-byte line.
template <class Store>
__device__ __forceinline__ int key_row(int place)
{
    return Store::kScaled ? place & 15 : (place & 4) << 1 | (place & 8) >> 1 | (place & 3);
}

template <class Store>
__host__ __device__ constexpr size_t cache_block_bytes(int page_size, int dim)
{
    return static_cast<size_t>(page_size) * (2 * dim * Store::kBytes + (Store::kScaled ? 2 : 0));
}

// Least exponent of an 8-bit row's scale.  Rows below 448 * 2^-110 keep it, so that no scale, inverse scale
// or code times scale is subnormal in fp32 (the smallest code is 2^-9).
constexpr int kLeastExponent = -110;

// The exponent e of a row's scale 2^e, biased by 127, from the bits of its largest finite magnitude:
// the least e with 448 * 2^e >= largest (448 = 1.75 * 2^8 is the largest e4m3 value).  A power of two makes
// the division exact and every stored value a bf16 number; it costs no precision, since e4m3 is a
// floating-point type itself.  Of the largest scale, 2^120, only codes up to 240 are used: 256 * 2^120 is no finite number.
constexpr uint32_t kLargestScale = 120 + 127, kCode240 = 0x77;
__device__ __forceinline__ uint32_t scale_byte(uint32_t largest_bits)
{
    const int e = static_cast<int>(largest_bits >> 23) - 127 - 8 + ((largest_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return static_cast<uint32_t>((e < kLeastExponent ? kLeastExponent : e) + 127);
}
__device__ __forceinline__ float scale_of(uint32_t byte) { return bits_to_f32(byte << 23); }

// Where a slot (page * page_size + place in the page) of head h lies; nullptr outside the pool.
struct PoolShape {
    PoolTable pool;
    uint32_t pages_per_rank, total_pages;
    int page_shift, heads;
    size_t block_bytes;
    __device__ __forceinline__ char *block(int64_t page, int h) const
    {
        if (page < 0 || page >= static_cast<int64_t>(total_pages)) return nullptr;
        const uint32_t p = static_cast<uint32_t>(page);
        const uint32_t rank = p / pages_per_rank, local = p - rank * pages_per_rank;
        return pool.p[rank] + (static_cast<size_t>(local) * heads + h) * block_bytes;
    }
};

// Checks a cache's description and fills in what the kernels take of it.
int check_cache(const tccl_paged_cache *cache, PoolShape *shape);

} // namespace tccl

// cache.hip -- the paged key/value cache that spans the ranks' buffers: tokens are written into it (in
// bf16, or in 8 bits with a power-of-two scale per token and head) and read back.  A slot is
// page * page_size + place in the page; pages are numbered over all ranks, rank r holding pages
// [r * pages_per_rank, (r + 1) * pages_per_rank).  The layout is described in rows.h.
//
// Both are moves: the floor is their bytes.  A workgroup takes 16 consecutive tokens of the list and one
// head, eight elements per lane (2 * head_dim lanes).  Keys go between rows and 16-byte chunks directly;
// values lie with their tokens innermost, so they pass through LDS, and what the workgroup's tokens do not
// cover of a 16-byte group is left to element stores (write) or read along (read).
#include "host.h"
#include "rows.h"

namespace tccl {

constexpr int kCacheTokens = 16;

struct CacheArgs {
    PoolShape shape;
    const int64_t *slots;
    size_t tokens;
    // write: strides of tokens and heads in bytes; read: contiguous [tokens][heads][head_dim]
    const char *k, *v;
    size_t k_token, k_head, v_token, v_head;
    char *k_out, *v_out;
};

// Largest finite magnitude of a lane's elements, as fp32 bits (order-preserving for magnitudes).
__device__ __forceinline__ float finite_magnitude(const float *x)
{
    float m = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float a = __builtin_fabsf(x[k]);
        m = fmaxf(m, __builtin_isfinite(a) ? a : 0.0f);
    }
    return m;
}

// Eight elements as they are stored: four dwords of bf16, or two of codes (and the row's scale byte).
template <class Store, int LANES>
__device__ __forceinline__ void encode(const float *x, uint32_t *code, uint32_t &scale)
{
    if constexpr (Store::kScaled) {
        scale = scale_byte(f32_to_bits(reduce_row<MaxOp, LANES>(finite_magnitude(x))));
        const float f = inverse_scale_of(scale);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            code[k] = pack_e4m3<false>(x[4 * k] * f, x[4 * k + 1] * f, 0);
            code[k] = pack_e4m3<true>(x[4 * k + 2] * f, x[4 * k + 3] * f, code[k]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) code[k] = pack_bf16(x[2 * k], x[2 * k + 1]);
    }
}

template <class Row, class Store, int LANES>
__global__ void __launch_bounds__(kCacheTokens * LANES)
cache_write_kernel(CacheArgs a)
{
    constexpr int D = 8 * LANES, BYTES = Store::kBytes, GROUP = Store::kChunk, CODES = 2 * BYTES;
    __shared__ __attribute__((aligned(16))) char values[kCacheTokens * D * BYTES];
    __shared__ char *block[kCacheTokens];  // of the token's page and this head, nullptr: not written
    __shared__ int place_in_page[kCacheTokens];
    const int h = blockIdx.y, t = threadIdx.x / LANES, p = threadIdx.x % LANES;
    const size_t first = static_cast<size_t>(blockIdx.x) * kCacheTokens;
    const int page_size = 1 << a.shape.page_shift;
    const size_t v_at = static_cast<size_t>(page_size) * D * BYTES, scales_at = 2 * v_at;
    if (threadIdx.x < kCacheTokens) {
        const size_t i = first + threadIdx.x;
        const int64_t slot = i < a.tokens ? a.slots[i] : -1;
        block[threadIdx.x] = slot < 0 ? nullptr : a.shape.block(slot >> a.shape.page_shift, h);
        place_in_page[threadIdx.x] = static_cast<int>(slot & (page_size - 1));
    }
    float k[8], v[8];
    if (first + t < a.tokens) {
        load_row<Row>(a.k + (first + t) * a.k_token + h * a.k_head + p * 8 * Row::kElemBytes, k);
        load_row<Row>(a.v + (first + t) * a.v_token + h * a.v_head + p * 8 * Row::kElemBytes, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) k[i] = v[i] = 0.0f;
    }
    __syncthreads();
    char *const mine = block[t];
    const int place = place_in_page[t];
    uint32_t code[CODES], k_scale = 0, v_scale = 0;
    encode<Store, LANES>(k, code, k_scale);
    if (mine != nullptr) {
        char *dst = mine + ((static_cast<size_t>(place >> 4) * (D / GROUP) + p * 8 / GROUP) * 16 + (place & 15)) * 16 +
                    (p * 8 % GROUP) * BYTES;
        if constexpr (Store::kScaled)
            *reinterpret_cast<u32x2 *>(dst) = u32x2{code[0], code[1]};
        else
            *reinterpret_cast<u32x4 *>(dst) = u32x4{code[0], code[1], code[2], code[3]};
    }
    encode<Store, LANES>(v, code, v_scale);
    {
        char *dst = values + (t * D + p * 8) * BYTES;
        if constexpr (Store::kScaled)
            *reinterpret_cast<u32x2 *>(dst) = u32x2{code[0], code[1]};
        else
            *reinterpret_cast<u32x4 *>(dst) = u32x4{code[0], code[1], code[2], code[3]};
    }
    if (Store::kScaled && mine != nullptr && p == 0) {
        mine[scales_at + place] = static_cast<char>(k_scale);
        mine[scales_at + page_size + place] = static_cast<char>(v_scale);
    }
    __syncthreads();
    // values: lane = dim, one group of GROUP tokens of the list at a time
    for (int item = threadIdx.x; item < D * (kCacheTokens / GROUP); item += kCacheTokens * LANES) {
        const int dim = item % D, t0 = item / D * GROUP;
        char *const b = block[t0];
        const int at = place_in_page[t0];
        bool whole = b != nullptr && at % GROUP == 0;
#pragma unroll
        for (int i = 1; i < GROUP; ++i) whole = whole && block[t0 + i] == b && place_in_page[t0 + i] == at + i;
        if (whole) {
            u32x4 out;
            if constexpr (Store::kScaled) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t u = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        u |= static_cast<uint32_t>(static_cast<uint8_t>(values[(t0 + 4 * i + j) * D + dim])) << (8 * j);
                    out[i] = u;
                }
            } else {
                const uint16_t *src = reinterpret_cast<const uint16_t *>(values) + t0 * D + dim;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    out[i] = static_cast<uint32_t>(src[2 * i * D]) | static_cast<uint32_t>(src[(2 * i + 1) * D]) << 16;
            }
            store_vec<false>(b + v_at, static_cast<size_t>(at / GROUP) * D + dim, out);
        } else {
            for (int i = 0; i < GROUP; ++i) {
                char *const bi = block[t0 + i];
                if (bi == nullptr) continue;
                const int pi = place_in_page[t0 + i];
                const size_t to = (static_cast<size_t>(pi / GROUP) * D + dim) * 16 + pi % GROUP * BYTES;
                if constexpr (Store::kScaled)
                    bi[v_at + to] = values[(t0 + i) * D + dim];
                else
                    *reinterpret_cast<uint16_t *>(bi + v_at + to) =
                        reinterpret_cast<const uint16_t *>(values)[(t0 + i) * D + dim];
            }
        }
    }
}

// Eight stored elements (codes of a row with one scale) in fp32.
template <class Store>
__device__ __forceinline__ void decode(const uint32_t *code, float scale, float *x)
{
    if constexpr (Store::kScaled) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            x[4 * k] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(code[k]), 0) * scale;
            x[4 * k + 1] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(code[k]), 1) * scale;
            x[4 * k + 2] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(code[k]), 2) * scale;
            x[4 * k + 3] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(code[k]), 3) * scale;
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            x[2 * k] = bits_to_f32(code[k] << 16);
            x[2 * k + 1] = bits_to_f32(code[k] & 0xFFFF0000u);
        }
    }
}

template <class Row, class Store, int LANES>
__global__ void __launch_bounds__(kCacheTokens * LANES)
cache_read_kernel(CacheArgs a)
{
    constexpr int D = 8 * LANES, BYTES = Store::kBytes, GROUP = Store::kChunk, CODES = 2 * BYTES;
    // one 16-byte value group per dim for each different group that the tokens lie in; a dim more per 16 keeps
    // the transposed reads off one bank
    __shared__ u32x4 groups[kCacheTokens][D];
    __shared__ const char *block[kCacheTokens];
    __shared__ int place_in_page[kCacheTokens], group_of[kCacheTokens], leader[kCacheTokens];
    __shared__ int count;
    const int h = blockIdx.y, t = threadIdx.x / LANES, p = threadIdx.x % LANES;
    const size_t first = static_cast<size_t>(blockIdx.x) * kCacheTokens;
    const int page_size = 1 << a.shape.page_shift;
    const size_t v_at = static_cast<size_t>(page_size) * D * BYTES, scales_at = 2 * v_at;
    if (threadIdx.x < 64) { // one whole wave: tokens are its first 16 lanes
        const size_t i = first + threadIdx.x;
        const int64_t slot = threadIdx.x < kCacheTokens && i < a.tokens ? a.slots[i] : -1;
        const char *b = slot < 0 ? nullptr : a.shape.block(slot >> a.shape.page_shift, h);
        const int place = static_cast<int>(slot & (page_size - 1));
        // a token leads a group unless the token before it lies in the same one
        const int64_t key = b == nullptr ? -1 : slot / GROUP;
        const int64_t before = __shfl_up(key, 1);
        const bool leads = key >= 0 && (threadIdx.x == 0 || before != key);
        const uint64_t mask = __ballot(leads);
        if (threadIdx.x < kCacheTokens) {
            block[threadIdx.x] = b;
            place_in_page[threadIdx.x] = place;
            const int n = __popcll(mask & ((2ull << threadIdx.x) - 1)) - 1;
            group_of[threadIdx.x] = n;
            if (leads) leader[n] = threadIdx.x;
        }
        if (threadIdx.x == 0) count = __popcll(mask);
    }
    __syncthreads();
    for (int item = threadIdx.x; item < count * D; item += kCacheTokens * LANES) {
        const int n = item / D, dim = item % D, l = leader[n];
        groups[n][dim] = load_vec<false>(block[l] + v_at, static_cast<size_t>(place_in_page[l] / GROUP) * D + dim);
    }
    const char *const mine = block[t];
    const int place = place_in_page[t];
    uint32_t code[CODES] = {};
    float k_scale = 0.0f, v_scale = 0.0f, x[8];
    if (mine != nullptr) {
        const char *src = mine +
                          ((static_cast<size_t>(place >> 4) * (D / GROUP) + p * 8 / GROUP) * 16 + (place & 15)) * 16 +
                          (p * 8 % GROUP) * BYTES;
#pragma unroll
        for (int i = 0; i < CODES; ++i) code[i] = reinterpret_cast<const uint32_t *>(src)[i];
        if constexpr (Store::kScaled) {
            k_scale = scale_of(static_cast<uint8_t>(mine[scales_at + place]));
            v_scale = scale_of(static_cast<uint8_t>(mine[scales_at + page_size + place]));
        }
    }
    const bool live = first + t < a.tokens;
    const size_t to = (((first + t) * a.shape.heads + h) * D + p * 8) * Row::kElemBytes;
    decode<Store>(code, k_scale, x);
    if (live) Row::store(a.k_out + to, x);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < CODES; ++i) code[i] = 0;
    if (mine != nullptr) {
        const int within = place % GROUP;
        const u32x4 *row = groups[group_of[t]];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (Store::kScaled)
                code[i >> 2] |= static_cast<uint32_t>(reinterpret_cast<const uint8_t *>(row + p * 8 + i)[within])
                                << (8 * (i & 3));
            else
                code[i >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(row + p * 8 + i)[within])
                                << (16 * (i & 1));
        }
    }
    decode<Store>(code, v_scale, x);
    if (live) Row::store(a.v_out + to, x);
}

static size_t block_bytes_of(const tccl_paged_cache &c)
{
    return c.dtype == TCCL_E4M3 ? cache_block_bytes<E4m3Store>(c.page_size, c.head_dim)
                                : cache_block_bytes<Bf16Store>(c.page_size, c.head_dim);
}

static int check_geometry(const tccl_paged_cache *c)
{
    if (c == nullptr || c->world < 1 || c->world > TCCL_MAX_WORLD) return TCCL_EINVAL;
    if (c->dtype != TCCL_BF16 && c->dtype != TCCL_E4M3) return TCCL_EINVAL;
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return TCCL_EINVAL;
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)) != 0) return TCCL_EINVAL;
    if (c->kv_heads < 1 || c->kv_heads > 65535) return TCCL_EINVAL;
    if (c->pages_per_rank < 1 || static_cast<int64_t>(c->pages_per_rank) * c->world > 0x7FFFFFFF) return TCCL_EINVAL;
    return TCCL_OK;
}

int check_cache(const tccl_paged_cache *c, PoolShape *shape)
{
    if (const int rc = check_geometry(c)) return rc;
    for (int i = 0; i < c->world; ++i) {
        if (c->bufs[i] == nullptr) return TCCL_EINVAL;
        if (!aligned16(c->bufs[i])) return TCCL_EALIGN;
        shape->pool.p[i] = static_cast<char *>(c->bufs[i]);
    }
    shape->pages_per_rank = static_cast<uint32_t>(c->pages_per_rank);
    shape->total_pages = static_cast<uint32_t>(c->pages_per_rank) * c->world;
    shape->page_shift = __builtin_ctz(c->page_size);
    shape->heads = c->kv_heads;
    shape->block_bytes = block_bytes_of(*c);
    return TCCL_OK;
}

template <class Row, class Store, int LANES>
static hipError_t launch_cache(bool write, const CacheArgs &a, hipStream_t stream)
{
    const dim3 grid(static_cast<unsigned>((a.tokens + kCacheTokens - 1) / kCacheTokens), a.shape.heads);
    if (write)
        hipLaunchKernelGGL((cache_write_kernel<Row, Store, LANES>), grid, dim3(kCacheTokens * LANES), 0, stream, a);
    else
        hipLaunchKernelGGL((cache_read_kernel<Row, Store, LANES>), grid, dim3(kCacheTokens * LANES), 0, stream, a);
    return hipGetLastError();
}

template <class Row, class Store>
static hipError_t launch_cache_dim(bool write, const CacheArgs &a, int dim, hipStream_t stream)
{
    switch (dim) {
    case 64: return launch_cache<Row, Store, 8>(write, a, stream);
    case 128: return launch_cache<Row, Store, 16>(write, a, stream);
    case 256: return launch_cache<Row, Store, 32>(write, a, stream);
    default: return hipErrorInvalidValue;
    }
}

static hipError_t launch_cache_types(bool write, const CacheArgs &a, const tccl_paged_cache &c, int dtype,
                                     hipStream_t stream)
{
    if (dtype == TCCL_BF16)
        return c.dtype == TCCL_E4M3 ? launch_cache_dim<Bf16Row, E4m3Store>(write, a, c.head_dim, stream)
                                    : launch_cache_dim<Bf16Row, Bf16Store>(write, a, c.head_dim, stream);
    return c.dtype == TCCL_E4M3 ? launch_cache_dim<F32Row, E4m3Store>(write, a, c.head_dim, stream)
                                : launch_cache_dim<F32Row, Bf16Store>(write, a, c.head_dim, stream);
}

constexpr size_t kMostTokens = static_cast<size_t>(1) << 31;

} // namespace tccl

using namespace tccl;

extern "C" size_t tccl_paged_cache_bytes(const tccl_paged_cache *cache)
{
    if (check_geometry(cache) != TCCL_OK) return 0;
    return static_cast<size_t>(cache->pages_per_rank) * cache->kv_heads * block_bytes_of(*cache);
}

extern "C" int tccl_cache_write(const tccl_paged_cache *cache, const void *k, const void *v, size_t k_token_stride,
                                size_t k_head_stride, size_t v_token_stride, size_t v_head_stride,
                                const int64_t *slots, size_t tokens, int dtype, void *stream)
{
    CacheArgs a = {};
    if (const int rc = check_cache(cache, &a.shape)) return rc;
    const size_t esize = dtype_size(dtype);
    if (esize == 0 || k == nullptr || v == nullptr || slots == nullptr || tokens > kMostTokens) return TCCL_EINVAL;
    if (!aligned16(k) || !aligned16(v)) return TCCL_EALIGN;
    a.k_token = k_token_stride * esize, a.k_head = k_head_stride * esize;
    a.v_token = v_token_stride * esize, a.v_head = v_head_stride * esize;
    if ((a.k_token | a.k_head | a.v_token | a.v_head) % kVecBytes != 0) return TCCL_EALIGN;
    if (tokens == 0) return TCCL_OK;
    a.slots = slots;
    a.tokens = tokens;
    a.k = static_cast<const char *>(k);
    a.v = static_cast<const char *>(v);
    return hip_code(launch_cache_types(true, a, *cache, dtype, static_cast<hipStream_t>(stream)));
}

extern "C" int tccl_cache_read(const tccl_paged_cache *cache, const int64_t *slots, size_t tokens, void *k_out,
                               void *v_out, int dtype, void *stream)
{
    CacheArgs a = {};
    if (const int rc = check_cache(cache, &a.shape)) return rc;
    if (dtype_size(dtype) == 0 || k_out == nullptr || v_out == nullptr || slots == nullptr || tokens > kMostTokens)
        return TCCL_EINVAL;
    if (!aligned16(k_out) || !aligned16(v_out)) return TCCL_EALIGN;
    if (tokens == 0) return TCCL_OK;
    a.slots = slots;
    a.tokens = tokens;
    a.k_out = static_cast<char *>(k_out);
    a.v_out = static_cast<char *>(v_out);
    return hip_code(launch_cache_types(false, a, *cache, dtype, static_cast<hipStream_t>(stream)));
}

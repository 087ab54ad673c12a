// cache.hip -- the paged key/value cache that spans the ranks' buffers: tokens are written into it (in
// bf16, or in 8 bits with a power-of-two scale per token and head) and read back.  A slot is
// page * page_size + place in the page; pages are numbered over all ranks, rank r holding pages
// [r * pages_per_rank, (r + 1) * pages_per_rank).  The layout is described in rows.h.
//
// Both are moves: the floor is their bytes.  A workgroup takes TOKENS (64; 16 of a short list) consecutive
// tokens of the list and one head.  Keys go between rows and 16-byte chunks directly.  Values lie with their tokens
// innermost, in 16-byte groups of 8 or 16 tokens per dim: the list is cut into runs, tokens that follow each other
// within one group, and a lane turns a run's 4 dims x 8 or 16 tokens in registers.  Reading takes a whole group and
// uses the run's part of it; writing stores whole groups with one store per dim, and of others (a run that begins or
// ends inside) what is whole of each four bytes, the rest element by element, since its neighbours may be
// written by another workgroup.
//
// Tokens that do not follow each other are runs of one: each of them reads its whole group, 8 or 16 times its values.
//
// 8 heads of 128, bf16 rows, in the kernel.  Reading 44,000 tokens: from 8 bits 49 to 58 us from process to process (4.7 to
// 5.6 TB/s, two thirds of it written), from bf16 73 us (5.0 TB/s).  Writing 8,192 of them that begin inside groups: in 8 bits 17.5 us
// (2.9 TB/s), in bf16 21.0 (3.2): a single residency of workgroups, in each of which loads, rounding, turning and stores
// follow each other; from a group's start 8,000 take 14.0 and 15.9 us where from inside one 17.9 and 19.2.
#include "host.h"
#include "rows.h"

namespace tccl {

constexpr int kCacheBlock = 256;

struct CacheArgs {
    PoolShape shape;
    const int64_t *slots;
    size_t tokens;
    // write: strides of tokens and heads in bytes; read: contiguous [tokens][heads][head_dim]
    const char *k, *v;
    size_t k_token, k_head, v_token, v_head;
    char *k_out, *v_out;
};

// Where the workgroup's tokens lie, and their runs.
template <int TOKENS>
struct Runs {
    char *block[TOKENS]; // of the token's page and this head, nullptr: outside the pool
    int place[TOKENS];   // in the page
    int first[TOKENS], length[TOKENS];
    int count;
};

// Run by the workgroup's first wave: lane i looks token i up.
template <int GROUP, int TOKENS>
__device__ __forceinline__ void find_runs(const CacheArgs &a, size_t begin, int h, Runs<TOKENS> &runs)
{
    const int lane = threadIdx.x;
    const int64_t slot = lane < TOKENS && begin + lane < a.tokens ? a.slots[begin + lane] : -1;
    char *const b = slot < 0 ? nullptr : a.shape.block(slot >> a.shape.page_shift, h);
    const int64_t before = __shfl_up(slot, 1);
    const bool live = b != nullptr;
    const bool leads = live && (lane == 0 || before + 1 != slot || slot % GROUP == 0);
    const uint64_t leaders = __ballot(leads), gaps = ~__ballot(live) | leaders;
    if (lane < TOKENS) {
        runs.block[lane] = b;
        runs.place[lane] = static_cast<int>(slot & ((1 << a.shape.page_shift) - 1));
    }
    if (leads) {
        const int n = __popcll(leaders & ((1ull << lane) - 1));
        const uint64_t behind = lane == 63 ? 0 : gaps >> (lane + 1); // the next leader or token without a place
        const int length = behind == 0 ? 64 - lane : __builtin_ctzll(behind) + 1;
        runs.first[n] = lane;
        runs.length[n] = length;
    }
    if (lane == 0) runs.count = __popcll(leaders);
}

// Four dwords as a 4 x 4 matrix of bytes, transposed.
__device__ __forceinline__ void transpose_bytes(uint32_t &a, uint32_t &b, uint32_t &c, uint32_t &d)
{
    const uint32_t ab_low = __builtin_amdgcn_perm(b, a, 0x05010400u), ab_high = __builtin_amdgcn_perm(b, a, 0x07030602u);
    const uint32_t cd_low = __builtin_amdgcn_perm(d, c, 0x05010400u), cd_high = __builtin_amdgcn_perm(d, c, 0x07030602u);
    a = __builtin_amdgcn_perm(cd_low, ab_low, 0x05040100u);
    b = __builtin_amdgcn_perm(cd_low, ab_low, 0x07060302u);
    c = __builtin_amdgcn_perm(cd_high, ab_high, 0x05040100u);
    d = __builtin_amdgcn_perm(cd_high, ab_high, 0x07060302u);
}

// A lane's part of a value group, 4 dims of GROUP tokens in 16 dwords: from by dim, as it is stored, to by token, or back
// (`TO_TOKENS` false).
template <class Store, bool TO_TOKENS>
__device__ __forceinline__ void turn_group(const uint32_t (&in)[16], uint32_t (&out)[16])
{
    if constexpr (Store::kScaled) { // 16 tokens: dim i is dwords 4 i ..., token t is dword t
#pragma unroll
        for (int q = 0; q < 4; ++q) { // tokens 4 q ... 4 q + 3
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = TO_TOKENS ? in[4 * i + q] : in[4 * q + i];
            transpose_bytes(w[0], w[1], w[2], w[3]);
#pragma unroll
            for (int i = 0; i < 4; ++i) out[TO_TOKENS ? 4 * q + i : 4 * i + q] = w[i];
        }
    } else { // 8 tokens: dim i is dwords 4 i ..., token t is dwords 2 t and 2 t + 1
#pragma unroll
        for (int q = 0; q < 4; ++q) // tokens 2 q and 2 q + 1
#pragma unroll
            for (int i = 0; i < 2; ++i) { // dims 2 i and 2 i + 1
                const int dim0 = 4 * (2 * i) + q, dim1 = 4 * (2 * i + 1) + q;
                const int token0 = 4 * q + i, token1 = 4 * q + 2 + i;
                const uint32_t x = in[TO_TOKENS ? dim0 : token0], y = in[TO_TOKENS ? dim1 : token1];
                out[TO_TOKENS ? token0 : dim0] = __builtin_amdgcn_perm(y, x, 0x05040100u);
                out[TO_TOKENS ? token1 : dim1] = __builtin_amdgcn_perm(y, x, 0x07060302u);
            }
    }
}

// Rows from here on take the path below: the fp32 bits of 1.9375 * 2^127, whose scale is 2^120 and whose code would round
// to 256, that is 2^128.
constexpr uint32_t kSpecialMagnitude = 0x7F780000u;

// A row with infinities, NaN or the largest finite numbers: its scale comes from the largest finite magnitude, what is not
// finite becomes NaN, and the codes of the largest scale stop at 240, so that no finite number becomes infinite.
template <class Row, int LANES>
__device__ __forceinline__ u32x2 codes_of_special_row(Row x, uint32_t &scale)
{
    constexpr uint32_t NOT_FINITE = 0x7F800000u;
    uint32_t largest = 0, nan = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const uint32_t u = f32_to_bits(x.at(k)) & 0x7FFFFFFFu;
        if (u >= NOT_FINITE)
            nan |= 1u << k;
        else
            largest = largest > u ? largest : u;
    }
    scale = scale_byte(f32_to_bits(reduce_row<MaxOp, LANES>(bits_to_f32(largest))));
    const u32x2 code = x.codes(scale_of(scale));
    u32x2 r = {0, 0};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        uint32_t c = (code[k >> 2] >> (8 * (k & 3))) & 0xFFu;
        if (scale == kLargestScale && (c & 0x7Fu) > kCode240) c = (c & 0x80u) | kCode240;
        if (nan & (1u << k)) c |= 0x7Fu;
        r[k >> 2] |= c << (8 * (k & 3));
    }
    return r;
}

// Eight elements as they are stored: four dwords of bf16, or two of codes (and the row's scale byte).
template <class Row, class Store, int LANES>
__device__ __forceinline__ void encode(const Row &x, char *to, uint32_t &scale)
{
    if constexpr (Store::kScaled) {
        const uint32_t m = x.magnitude();
        u32x2 code;
        if (__any(m >= kSpecialMagnitude)) {
            code = codes_of_special_row<Row, LANES>(x, scale);
        } else {
            scale = scale_byte(f32_to_bits(reduce_row<MaxOp, LANES>(bits_to_f32(m))));
            code = x.codes(scale_of(scale));
        }
        if (to != nullptr) *reinterpret_cast<u32x2 *>(to) = code;
    } else if (to != nullptr) {
        float f[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = x.at(k);
        Bf16Row::store(to, f);
    }
}

template <class Row, class Store, int LANES, int TOKENS>
__global__ void __launch_bounds__(kCacheBlock)
cache_write_kernel(CacheArgs a)
{
    constexpr int D = 8 * LANES, BYTES = Store::kBytes, GROUP = Store::kChunk, IN_DWORD = 4 / BYTES;
    constexpr int ROUNDS = (TOKENS * LANES + kCacheBlock - 1) / kCacheBlock;
    __shared__ __attribute__((aligned(16))) char values[TOKENS * D * BYTES];
    __shared__ Runs<TOKENS> runs;
    const int h = blockIdx.y, p = threadIdx.x % LANES;
    const size_t begin = static_cast<size_t>(blockIdx.x) * TOKENS;
    const int page_size = 1 << a.shape.page_shift;
    const size_t v_at = static_cast<size_t>(page_size) * D * BYTES, scales_at = 2 * v_at;
    Row k[ROUNDS], v[ROUNDS];
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        const int t = (threadIdx.x + i * kCacheBlock) / LANES;
        if (t < TOKENS && begin + t < a.tokens) {
            k[i].load(a.k + (begin + t) * a.k_token + h * a.k_head + p * 8 * Row::kElemBytes);
            v[i].load(a.v + (begin + t) * a.v_token + h * a.v_head + p * 8 * Row::kElemBytes);
        } else {
            k[i].zero();
            v[i].zero();
        }
    }
    if (threadIdx.x < 64) find_runs<GROUP, TOKENS>(a, begin, h, runs);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        const int t = (threadIdx.x + i * kCacheBlock) / LANES;
        if (t >= TOKENS) break; // whole waves
        char *const block = runs.block[t];
        const int place = runs.place[t];
        uint32_t k_scale = 0, v_scale = 0;
        const size_t chunk = static_cast<size_t>(place >> 4) * (D / GROUP) + p * 8 / GROUP;
        encode<Row, Store, LANES>(
            k[i], block == nullptr ? nullptr : block + (chunk * 16 + key_row<Store>(place)) * 16 + (p * 8 % GROUP) * BYTES, k_scale);
        encode<Row, Store, LANES>(v[i], values + (t * D + p * 8) * BYTES, v_scale);
        if (Store::kScaled && block != nullptr && p == 0) {
            block[scales_at + place] = static_cast<char>(k_scale);
            block[scales_at + page_size + place] = static_cast<char>(v_scale);
        }
    }
    __syncthreads();
    for (int item = threadIdx.x; item < runs.count * (D / 4); item += kCacheBlock) {
        const int n = item / (D / 4), dim = item % (D / 4) * 4;
        const int first = runs.first[n], length = runs.length[n], place = runs.place[first], start = place % GROUP;
        uint32_t by_token[16], by_dim[16];
#pragma unroll
        for (int t = 0; t < GROUP; ++t) {
            // tokens of the group that are not in the run: any of its own, which are not stored there
            const int at = first + (t < start ? 0 : (t < start + length ? t - start : length - 1));
            const char *src = values + (at * D + dim) * BYTES;
#pragma unroll
            for (int w = 0; w < BYTES; ++w) by_token[t * BYTES + w] = reinterpret_cast<const uint32_t *>(src)[w];
        }
        turn_group<Store, false>(by_token, by_dim);
        char *const to = runs.block[first] + v_at + (static_cast<size_t>(place / GROUP) * D + dim) * 16;
        if (length == GROUP) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                store_vec<false>(to, i, u32x4{by_dim[4 * i], by_dim[4 * i + 1], by_dim[4 * i + 2], by_dim[4 * i + 3]});
            continue;
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int low = w * IN_DWORD; // the dword's first token
            if (low >= start && low + IN_DWORD <= start + length) {
#pragma unroll
                for (int i = 0; i < 4; ++i) *reinterpret_cast<uint32_t *>(to + i * 16 + w * 4) = by_dim[4 * i + w];
                continue;
            }
#pragma unroll
            for (int t = 0; t < IN_DWORD; ++t) {
                if (low + t < start || low + t >= start + length) continue;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t x = by_dim[4 * i + w] >> (8 * BYTES * t);
                    if constexpr (Store::kScaled)
                        to[i * 16 + low + t] = static_cast<char>(x);
                    else
                        *reinterpret_cast<uint16_t *>(to + i * 16 + (low + t) * 2) = static_cast<uint16_t>(x);
                }
            }
        }
    }
}

// N (4 or 8) stored elements of a row with one scale, in fp32.
template <class Store, int N>
__device__ __forceinline__ void decode(const uint32_t *code, float scale, float *x)
{
    if constexpr (Store::kScaled) {
#pragma unroll
        for (int k = 0; k < N / 4; ++k) {
            const f32x2 low = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(code[k]), false);
            const f32x2 high = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(code[k]), true);
            x[4 * k] = low.x * scale;
            x[4 * k + 1] = low.y * scale;
            x[4 * k + 2] = high.x * scale;
            x[4 * k + 3] = high.y * scale;
        }
    } else {
#pragma unroll
        for (int k = 0; k < N / 2; ++k) {
            x[2 * k] = bits_to_f32(code[k] << 16);
            x[2 * k + 1] = bits_to_f32(code[k] & 0xFFFF0000u);
        }
    }
}

// Four elements of a row.
template <class Row>
__device__ __forceinline__ void store_four(char *to, const float *x)
{
    if constexpr (Row::kElemBytes == 2)
        *reinterpret_cast<u32x2 *>(to) = u32x2{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
    else
        store_vec<false>(to, 0, u32x4{f32_to_bits(x[0]), f32_to_bits(x[1]), f32_to_bits(x[2]), f32_to_bits(x[3])});
}

template <class Row, class Store, int LANES, int TOKENS>
__global__ void __launch_bounds__(kCacheBlock)
cache_read_kernel(CacheArgs a)
{
    constexpr int D = 8 * LANES, BYTES = Store::kBytes, GROUP = Store::kChunk, CODES = 2 * BYTES;
    constexpr int ROUNDS = (TOKENS * LANES + kCacheBlock - 1) / kCacheBlock;
    typedef uint32_t codes_t __attribute__((ext_vector_type(CODES)));
    __shared__ Runs<TOKENS> runs;
    const int h = blockIdx.y;
    const size_t begin = static_cast<size_t>(blockIdx.x) * TOKENS;
    const int page_size = 1 << a.shape.page_shift;
    const size_t v_at = static_cast<size_t>(page_size) * D * BYTES, scales_at = 2 * v_at;
    const size_t token_bytes = static_cast<size_t>(a.shape.heads) * D * Row::kElemBytes;
    const size_t to = begin * token_bytes + static_cast<size_t>(h) * D * Row::kElemBytes;
    if (threadIdx.x < 64) find_runs<GROUP, TOKENS>(a, begin, h, runs);
    __syncthreads();
    const int here = a.tokens - begin < TOKENS ? static_cast<int>(a.tokens - begin) : TOKENS;
    codes_t k[ROUNDS]; // eight elements of a row per lane, as the stores want them
    uint32_t k_scale[ROUNDS];
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        const int t = (threadIdx.x + i * kCacheBlock) / LANES, p = (threadIdx.x + i * kCacheBlock) % LANES;
        k[i] = codes_t(0);
        k_scale[i] = 0;
        if (t >= here) continue;
        const char *const block = runs.block[t];
        const int place = runs.place[t];
        if (block == nullptr) continue;
        const size_t chunk = static_cast<size_t>(place >> 4) * (D / GROUP) + p * 8 / GROUP;
        k[i] = *reinterpret_cast<const codes_t *>(block + (chunk * 16 + key_row<Store>(place)) * 16 + (p * 8 % GROUP) * BYTES);
        if constexpr (Store::kScaled) k_scale[i] = static_cast<uint8_t>(block[scales_at + place]);
    }
    for (int item = threadIdx.x; item < runs.count * (D / 4); item += kCacheBlock) {
        const int n = item / (D / 4), dim = item % (D / 4) * 4;
        const int first = runs.first[n], length = runs.length[n], place = runs.place[first], start = place % GROUP;
        const char *const from = runs.block[first] + v_at + (static_cast<size_t>(place / GROUP) * D + dim) * 16;
        uint32_t by_dim[16], by_token[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const u32x4 u = load_vec<false>(from, i);
#pragma unroll
            for (int w = 0; w < 4; ++w) by_dim[4 * i + w] = u[w];
        }
        u32x4 scales = {};
        if constexpr (Store::kScaled)
            scales = load_vec<false>(runs.block[first] + scales_at + page_size + (place - start), 0);
        turn_group<Store, true>(by_dim, by_token);
        char *const out = a.v_out + to + dim * Row::kElemBytes;
#pragma unroll
        for (int t = 0; t < GROUP; ++t) {
            if (t < start || t >= start + length) continue;
            float x[4];
            decode<Store, 4>(by_token + t * BYTES, scale_of((scales[(t >> 2) & 3] >> (8 * (t & 3))) & 0xFFu), x);
            store_four<Row>(out + (first + t - start) * token_bytes, x);
        }
    }
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        const int t = (threadIdx.x + i * kCacheBlock) / LANES, p = (threadIdx.x + i * kCacheBlock) % LANES;
        if (t >= here) continue;
        uint32_t code[CODES];
#pragma unroll
        for (int w = 0; w < CODES; ++w) code[w] = k[i][w];
        const size_t at = to + t * token_bytes + p * 8 * Row::kElemBytes;
        float x[8];
        decode<Store, 8>(code, scale_of(k_scale[i]), x);
        Row::store(a.k_out + at, x);
        if (runs.block[t] == nullptr) { // no run: the token's values are zeros as well
            const float zeros[8] = {};
            Row::store(a.v_out + at, zeros);
        }
    }
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
    // below 2^47 blocks, of up to 2^18 bytes: a buffer's size has to fit its type
    const size_t blocks = static_cast<size_t>(c->pages_per_rank) * c->kv_heads;
    return blocks <= static_cast<size_t>(PTRDIFF_MAX) / block_bytes_of(*c) ? TCCL_OK : TCCL_EINVAL;
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

template <class Row, class Store, int LANES, int TOKENS>
static hipError_t launch_cache_tokens(bool write, const CacheArgs &a, hipStream_t stream)
{
    const dim3 grid(static_cast<unsigned>((a.tokens + TOKENS - 1) / TOKENS), a.shape.heads);
    if (write)
        hipLaunchKernelGGL((cache_write_kernel<Row, Store, LANES, TOKENS>), grid, dim3(kCacheBlock), 0, stream, a);
    else
        hipLaunchKernelGGL((cache_read_kernel<Row, Store, LANES, TOKENS>), grid, dim3(kCacheBlock), 0, stream, a);
    return hipGetLastError();
}

// Tiles of 64 tokens where they fill the GPU twice, else of 16.  8 heads of 128 in 8 bits, write and read of tokens from a
// group's start: 1,000 tokens 6.1 and 5.7 us with 64, 4.9 and 5.1 with 16; 4,000 9.4 and 8.1 against 9.5 and 7.8; 8,000 14.0 and
// 10.2 against 14.2 and 12.5.  Written from inside a group, where smaller tiles cut more runs: 6.8 against 7.0, 11.6 against
// 17.5, 17.9 against 27.8.
template <class Row, class Store, int LANES>
static hipError_t launch_cache(bool write, const CacheArgs &a, hipStream_t stream)
{
    if (a.tokens / 64 * a.shape.heads >= static_cast<size_t>(compute_units()) * 2)
        return launch_cache_tokens<Row, Store, LANES, 64>(write, a, stream);
    return launch_cache_tokens<Row, Store, LANES, 16>(write, a, stream);
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

constexpr size_t kMostTokens = static_cast<size_t>(1) << 29; // as many tiles of 64 are one launch

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

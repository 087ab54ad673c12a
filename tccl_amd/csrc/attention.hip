// attention.hip -- attention of one new token per sequence over the paged cache of all ranks, split over the
// cache's length and joined; and the softmax-weighted all-reduce that joins the ranks' own partial
// attentions.
//
//   o = sum_t p_t v_t / sum_t p_t,  p_t = exp(s_t - m),  s_t = scale q.k_t,  m = max_t s_t,  lse = m + log sum_t p_t
// A part of the tokens gives (m, l = sum p, O = sum p v) with its own m; parts join by
//   m = max m_i,  l = sum l_i exp(m_i - m),  O = sum O_i exp(m_i - m)
// in any grouping.  No tokens give o = 0 and lse = -inf.
//
// The cache is read once; that is the floor, and HBM the bound: 64 sequences of 2,048 to 8,192 tokens of 8 key heads
// of 128 in 8 bits take 117 us in the kernel, 5.8 TB/s (a large sum of torch reads at 6.2), with vector instructions a
// third and matrix instructions a tenth of the time.  Scores come as S^T = K Q^T and the output as
// O^T = V^T P^T from 16x16x32 matrix instructions: the cache's layout makes every 16-byte load an operand as it stands,
// and a lane's scores are the tokens that the lane holds of P, so nothing passes through LDS and a query head's
// running maximum and sum stay with one lane column.  The next block's keys are loaded once the scores are formed and
// its values once this block's are used, into the same registers, so that loads are always on their way.
#include "host.h"
#include "rows.h"

namespace tccl {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kAttnBlock = 256;
constexpr int kAttnWaves = 4;
constexpr int kPiecePages = 512;  // page addresses a workgroup looks up at once
constexpr size_t kBatch = 4096;  // sequences of a launch at most: every workgroup adds their lengths up
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

struct AttnArgs {
    PoolShape shape;
    const char *q;
    size_t q_batch, q_head; // bytes
    const int32_t *table;
    size_t table_row;       // elements
    const int32_t *lengths;
    char *out;
    float *lse;             // may be nullptr
    float *part_o, *part_ml; // [workgroups][2][heads of a workgroup][D] and [..][2]: see decode_attention_kernel
    int2 *spans;            // [batch * head_groups]: a row's first partial and how many workgroups it spans
    int batch, q_heads, group; // query heads: all, and per key head
    int blocks_per_wg, head_groups; // blocks of 16 query heads in a workgroup (1, 2, 4); rows per sequence
    int most;               // tokens of a sequence at most
    int workgroups;         // that share the tokens; 0: a workgroup per row
    float scale;            // times log2(e)
};

__device__ __forceinline__ bf16x8 as_operand(u32x4 v) { return __builtin_bit_cast(bf16x8, v); }

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_operand(a), as_operand(b), c, 0, 0, 0);
}

// Eight e4m3 codes as eight bf16 numbers (exact).
__device__ __forceinline__ u32x4 widen_e4m3(uint32_t lo, uint32_t hi)
{
    u32x4 r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
    return r;
}

__device__ __forceinline__ int sequence_length(const AttnArgs &a, int b)
{
    const int n = a.lengths[b];
    return n < 0 ? 0 : (n < a.most ? n : a.most);
}

// Dealing out `units` to `workgroups`: the first `rest` of them get one more than the others.
struct Shares {
    uint32_t each, rest;
    __device__ __forceinline__ Shares(uint32_t units, uint32_t workgroups)
        : each(units / workgroups), rest(units - each * workgroups)
    {
    }
    __device__ __forceinline__ uint32_t begin(uint32_t w) const { return w * each + (w < rest ? w : rest); }
    __device__ __forceinline__ uint32_t owner(uint32_t unit) const
    {
        const uint32_t longer = rest * (each + 1);
        return unit < longer ? unit / (each + 1) : rest + (unit - longer) / each;
    }
};

// Exclusive prefix sum over the workgroup's threads; `total` is the sum.
__device__ __forceinline__ uint32_t prefix_sum(uint32_t x, uint32_t *wave_sums, uint32_t &total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t sum = x;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
        const uint32_t up = __shfl_up(sum, step);
        sum += lane >= step ? up : 0;
    }
    if (lane == 63) wave_sums[wave] = sum;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kAttnWaves; ++w) {
        before += w < wave ? wave_sums[w] : 0;
        total += wave_sums[w];
    }
    return before + sum - x;
}

// A row is a sequence, a key head and up to 64 of the query heads that share it (blocks of 16); its tokens are
// cut into units of four token blocks.  All rows' units, one row behind the other, are dealt out evenly to the
// workgroups, so that ragged lengths leave no workgroup with more than its share.  A row that lies in one
// workgroup is finished there.  Of the others each workgroup leaves its part of (m, l, O): in place 0 the row
// that holds its first unit, in place 1 the row that it begins and does not end; join_parts_kernel
// joins them.  Four waves: blocks_per_wg of them work on different blocks of query heads and the same
// tokens (which they share through the caches), the others on different tokens.
//
// Lane layout, lane = 16 g + m:
//   K operand    row m is a token, the lane's 16 bytes are its dims 16-byte chunk g of four
//   Q operand    column m is a query head, the same dims
//   S^T          column m is the query head, rows 4 g + i
//   V^T operand  row m is a dim, the lane's 16 bytes are tokens of group g
//   P^T operand  column m is the query head, the same tokens
// A block is four groups of TOKENS = 8 (bf16) or 16 (8 bits) consecutive tokens.  Row 4 g + i of the block's
// K tile t is token TOKENS g + 4 t + i, so that S^T leaves the tokens of group g in lanes 16 g ... 16 g + 15,
// where P^T needs them.
template <class Store, int D, bool NT>
__global__ void __launch_bounds__(kAttnBlock, D == 256 ? 1 : 2)
decode_attention_kernel(AttnArgs a)
{
    constexpr int TOKENS = Store::kChunk, TILES = TOKENS / 4, BLOCK = 4 * TOKENS, UNIT = kAttnWaves * BLOCK;
    constexpr int KLOADS = D / (4 * Store::kChunk);          // 16-byte chunks of a token's row per lane
    constexpr int QSTEPS = D / 32, DTILES = D / 16, PARTS = TOKENS / 8;
    __shared__ const char *pages[kPiecePages];
    __shared__ float wave_m[kAttnWaves][16], wave_l[kAttnWaves][16];
    __shared__ float wave_o[kAttnWaves][16][D + 4];
    __shared__ uint32_t wave_sums[kAttnWaves], found[3];

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, m = lane & 15;
    const int shift = a.shape.page_shift, page_size = 1 << shift;
    const size_t v_at = static_cast<size_t>(page_size) * D * Store::kBytes;
    const char *const safe = a.shape.pool.p[0]; // read, and masked, where there is no page
    const int my_block = wave % a.blocks_per_wg, my_turn = wave / a.blocks_per_wg, turns = kAttnWaves / a.blocks_per_wg;

    // the workgroup's units [unit, stop) of all, and the row that `unit` lies in
    uint32_t unit, stop, row_begin; // row_begin: the first unit of the row
    int b, hg, length;
    Shares shares(0, 1);
    if (a.workgroups == 0) {
        b = blockIdx.x / a.head_groups;
        hg = blockIdx.x % a.head_groups;
        length = sequence_length(a, b);
        unit = row_begin = 0;
        stop = (length + UNIT - 1) / UNIT;
        if (length == 0) stop = 1; // an empty row: one pass over no tokens, which writes its zeros
    } else {
        const int per = (a.batch + kAttnBlock - 1) / kAttnBlock, first = threadIdx.x * per;
        const int last = first + per < a.batch ? first + per : a.batch;
        uint32_t mine = 0;
        for (int i = first; i < last; ++i) mine += (sequence_length(a, i) + UNIT - 1) / UNIT;
        uint32_t all;
        uint32_t before = prefix_sum(mine, wave_sums, all);
        shares = Shares(all * a.head_groups, gridDim.x);
        unit = shares.begin(blockIdx.x);
        stop = shares.begin(blockIdx.x + 1);
        if (unit < stop && unit >= before * a.head_groups && unit < (before + mine) * a.head_groups) {
            for (int i = first; i < last; ++i) {
                const int n = sequence_length(a, i);
                const uint32_t units = (n + UNIT - 1) / UNIT;
                if (unit < (before + units) * a.head_groups) {
                    found[0] = i;
                    found[1] = before * a.head_groups;
                    found[2] = n;
                    break;
                }
                before += units;
            }
        }
        // rows without tokens have no units: their zeros are written here
        for (int e = blockIdx.x; e < a.batch; e += gridDim.x) {
            if (sequence_length(a, e) > 0) continue;
            const size_t row = static_cast<size_t>(e) * a.q_heads;
            for (int i = threadIdx.x; i < a.q_heads * (D / 8); i += kAttnBlock)
                store_vec<false>(a.out + row * D * 2, i, u32x4{0, 0, 0, 0});
            for (int i = threadIdx.x; i < a.q_heads; i += kAttnBlock)
                if (a.lse != nullptr) a.lse[row + i] = -__builtin_inff();
            for (int i = threadIdx.x; i < a.head_groups; i += kAttnBlock) a.spans[e * a.head_groups + i] = int2{0, 0};
        }
        if (unit == stop) return;
        __syncthreads();
        b = found[0];
        length = found[2];
        const uint32_t n = (length + UNIT - 1) / UNIT;
        hg = (unit - found[1]) / n;
        row_begin = found[1] + hg * n;
    }

    for (bool first_row = true; unit < stop; first_row = false) {
        const uint32_t row_units = length == 0 ? 1 : (length + UNIT - 1) / UNIT;
        const uint32_t row_end = row_begin + row_units, until = row_end < stop ? row_end : stop;
        const int groups_per_head = a.head_groups / a.shape.heads;
        const int h = hg / groups_per_head, first_of_group = hg % groups_per_head * a.blocks_per_wg * 16;
        const int left = a.group - first_of_group, in_wg = left < 16 * a.blocks_per_wg ? left : 16 * a.blocks_per_wg;
        const int first_head = h * a.group + first_of_group; // of the workgroup's in_wg query heads
        const int in_block = in_wg - 16 * my_block;          // of the wave's, may be over 16 or below 1

        u32x4 q[QSTEPS];
#pragma unroll
        for (int s = 0; s < QSTEPS; ++s) {
            // the dims of contraction step s that lane group g holds
            const int dim = Store::kScaled ? (s >> 1) * 64 + g * 16 + (s & 1) * 8 : s * 32 + g * 8;
            q[s] = u32x4{0, 0, 0, 0};
            if (m < in_block)
                q[s] = load_vec<false>(
                    a.q + b * a.q_batch + (first_head + 16 * my_block + m) * a.q_head + dim * 2, 0);
        }
        float top = -__builtin_inff(), total = 0.0f;
        f32x4 acc[DTILES];
#pragma unroll
        for (int i = 0; i < DTILES; ++i) acc[i] = f32x4{0, 0, 0, 0};

        const int row_stop = static_cast<int>(until - row_begin) * UNIT < length
                                 ? static_cast<int>(until - row_begin) * UNIT
                                 : length;
        for (int begin = static_cast<int>(unit - row_begin) * UNIT; begin < row_stop;) {
            // a piece: what kPiecePages pages cover, in whole units
            const int first_page = begin >> shift;
            const int reach = ((first_page + kPiecePages) << shift) / UNIT * UNIT;
            const int end = reach < row_stop && reach > 0 ? reach : row_stop;
            const int npages = ((end - 1) >> shift) - first_page + 1;
            __syncthreads();
            for (int i = threadIdx.x; i < npages; i += kAttnBlock)
                pages[i] = a.shape.block(a.table[static_cast<size_t>(b) * a.table_row + first_page + i], h);
            __syncthreads();

            u32x4 k[TILES][KLOADS], v[DTILES], k_scales = {}, v_scales = {};
            // lane m's token of tile t lies in group m / 4 of the block
            auto load_keys = [&](int start) {
                const int at = start + (m >> 2) * TOKENS, p = (at >> shift) - first_page;
                const char *kb = p < npages ? pages[p] : nullptr;
                kb = kb != nullptr ? kb : safe;
                const int in = at & (page_size - 1), first = key_row<Store>(in) + (m & 3);
                const char *row = kb + static_cast<size_t>(in >> 4) * (D / Store::kChunk) * 256 + first * 16 + g * 256;
                // token 4 t of a group is key_row(4 t) = 4 t rows (8 bits) or 8 t rows on.  Tiles innermost: they share cache
                // lines in 8 bits
                constexpr int TILE_BYTES = Store::kScaled ? 64 : 128;
#pragma unroll
                for (int c = 0; c < KLOADS; ++c)
#pragma unroll
                    for (int t = 0; t < TILES; ++t) k[t][c] = load_vec<NT>(row + c * 1024 + t * TILE_BYTES, 0);
            };
            // values and scores: group g.  `live`: the tokens of it that count
            int live = 0;
            auto load_values = [&](int start) {
                const int at = start + g * TOKENS, p = (at >> shift) - first_page;
                const char *vb = p < npages ? pages[p] : nullptr;
                live = vb != nullptr ? end - at : 0;
                vb = vb != nullptr ? vb : safe;
                const int in = at & (page_size - 1);
#pragma unroll
                for (int d = 0; d < DTILES; ++d)
                    v[d] = load_vec<NT>(vb + v_at + (static_cast<size_t>(in / TOKENS) * D + d * 16 + m) * 16, 0);
                if constexpr (Store::kScaled) {
                    k_scales = load_vec<false>(vb + 2 * v_at + in, 0);
                    v_scales = load_vec<false>(vb + 2 * v_at + page_size + in, 0);
                }
            };
            int start = begin + my_turn * BLOCK;
            if (start < end) {
                load_keys(start);
                load_values(start);
            }
            for (; start < end; start += turns * BLOCK) {
                const int next = start + turns * BLOCK;
                f32x4 s[TILES];
#pragma unroll
                for (int t = 0; t < TILES; ++t) s[t] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < KLOADS; ++i) // tiles innermost: their chains of products do not wait for each other
#pragma unroll
                    for (int half = 0; half < (Store::kScaled ? 2 : 1); ++half)
#pragma unroll
                        for (int t = 0; t < TILES; ++t) {
                            if constexpr (Store::kScaled)
                                s[t] = mfma(widen_e4m3(k[t][i][2 * half], k[t][i][2 * half + 1]), q[2 * i + half], s[t]);
                            else
                                s[t] = mfma(k[t][i], q[i], s[t]);
                        }
                if (next < end) load_keys(next);
#pragma unroll
                for (int t = 0; t < TILES; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float x = s[t][i] * a.scale;
                        if constexpr (Store::kScaled) x = x * scale_of((k_scales[t] >> (8 * i)) & 0xFFu);
                        s[t][i] = 4 * t + i < live ? x : -__builtin_inff();
                    }
                float best = s[0][0];
#pragma unroll
                for (int t = 0; t < TILES; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) best = fmaxf(best, s[t][i]);
                best = across32<MaxOp>(across16<MaxOp>(best));
                if (__any(best > top)) {
                    const float higher = fmaxf(top, best);
                    const float f = higher == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(top - higher);
                    top = higher;
                    total = total * f;
#pragma unroll
                    for (int d = 0; d < DTILES; ++d) acc[d] = acc[d] * f;
                }
                const float from = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
                for (int t = 0; t < TILES; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p = __builtin_amdgcn_exp2f(s[t][i] - from);
                        total = total + p;
                        s[t][i] = p;
                        if constexpr (Store::kScaled)
                            s[t][i] = 4 * t + i < live ? p * scale_of((v_scales[t] >> (8 * i)) & 0xFFu) : 0.0f;
                    }
                if (!__all(live >= TOKENS)) { // what lies behind the last token may be anything, NaN too
                    constexpr int EACH = 4 / Store::kBytes;
#pragma unroll
                    for (int d = 0; d < DTILES; ++d)
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const int in_word = live - w * EACH;
                            v[d][w] &= in_word >= EACH ? ~0u
                                                       : (in_word <= 0 ? 0u : (1u << (8 * Store::kBytes * in_word)) - 1u);
                        }
                }
#pragma unroll
                for (int part = 0; part < PARTS; ++part) {
                    // P in two bf16 terms, so that its rounding (2^-9 of each weight) does not reach the output
                    u32x4 hi, lo;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const float x = s[2 * part + (w >> 1)][(2 * w) & 3], y = s[2 * part + (w >> 1)][(2 * w + 1) & 3];
                        hi[w] = pack_bf16(x, y);
                        lo[w] = pack_bf16(x - bits_to_f32(hi[w] << 16), y - bits_to_f32(hi[w] & 0xFFFF0000u));
                    }
#pragma unroll
                    for (int d = 0; d < DTILES; ++d) {
                        u32x4 vd;
                        if constexpr (Store::kScaled)
                            vd = widen_e4m3(v[d][2 * part], v[d][2 * part + 1]);
                        else
                            vd = v[d];
                        acc[d] = mfma(vd, hi, acc[d]);
                        acc[d] = mfma(vd, lo, acc[d]);
                    }
                }
                if (next < end) load_values(next);
            }
            begin = end;
        }

        // the waves' parts: lane groups hold the sums of their own tokens, and all dims of O
        total = across32<AddOp>(across16<AddOp>(total));
        __syncthreads();
        if (g == 0) {
            wave_m[wave][m] = top;
            wave_l[wave][m] = total;
        }
#pragma unroll
        for (int d = 0; d < DTILES; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) wave_o[wave][m][d * 16 + 4 * g + i] = acc[d][i];
        __syncthreads();
        const bool whole = unit == row_begin && until == row_end;
        const size_t part = 2 * blockIdx.x + (first_row ? 0 : 1);
        for (int item = threadIdx.x; item < in_wg * (D / 4); item += kAttnBlock) {
            const int n = item / (D / 4), d = item % (D / 4) * 4, block = n >> 4, at = n & 15;
            float best = -__builtin_inff();
            for (int w = block; w < kAttnWaves; w += a.blocks_per_wg) best = fmaxf(best, wave_m[w][at]);
            const float from = best == -__builtin_inff() ? 0.0f : best;
            float l = 0.0f;
            f32x4 o = {0, 0, 0, 0};
            for (int w = block; w < kAttnWaves; w += a.blocks_per_wg) {
                const float f = __builtin_amdgcn_exp2f(wave_m[w][at] - from);
                l = __builtin_fmaf(wave_l[w][at], f, l);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = __builtin_fmaf(wave_o[w][at][d + i], f, o[i]);
            }
            if (whole) {
                const size_t row = static_cast<size_t>(b) * a.q_heads + first_head + n;
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                *reinterpret_cast<u32x2 *>(a.out + (row * D + d) * 2) =
                    u32x2{pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv)};
                if (d == 0 && a.lse != nullptr)
                    a.lse[row] = l == 0.0f ? -__builtin_inff() : (best + __builtin_amdgcn_logf(l)) * kLn2;
            } else {
                const size_t to = part * (16 * a.blocks_per_wg) + n;
                *reinterpret_cast<f32x4 *>(a.part_o + to * D + d) = o;
                if (d == 0) {
                    a.part_ml[2 * to] = best;
                    a.part_ml[2 * to + 1] = l;
                }
            }
        }
        if (a.workgroups == 0) return;
        if (unit == row_begin && threadIdx.x == 0)
            a.spans[b * a.head_groups + hg] =
                int2{static_cast<int>(part), static_cast<int>(shares.owner(row_end - 1) - blockIdx.x) + 1};
        // the next row
        unit = until;
        row_begin = row_end;
        if (++hg == a.head_groups) {
            hg = 0;
            if (unit < stop) // there is a next row with tokens
                do length = sequence_length(a, ++b);
                while (length == 0 && b + 1 < a.batch);
        }
    }
}

// WAVES waves per (sequence, query head) that spans several workgroups, each taking every WAVES-th part: its lanes weigh
// up to 64 of them at a time, then it adds them up, D / 64 dims per lane, with FLIGHT parts' loads in flight; a
// part's weight reaches the other lanes through a scalar register.  (4,096 rows of two or three parts 4.9 us with four in flight,
// 5.9 with 16; 72 rows of 85 parts 9 with eight, 8 with 16, 11 with 32.)
template <int D, int WAVES>
__global__ void __launch_bounds__(256)
join_parts_kernel(AttnArgs a)
{
    constexpr int EACH = D / 64, FLIGHT = WAVES == 1 ? 4 : 16;
    typedef float part_t __attribute__((ext_vector_type(EACH)));
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, mine = WAVES == 1 ? 0 : wave;
    const int row = WAVES == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
    if (row >= a.batch * a.q_heads) return;
    const int b = row / a.q_heads, head = row - b * a.q_heads;
    const int wide = 16 * a.blocks_per_wg, h = head / a.group, in_group = head - h * a.group;
    const int hg = h * (a.head_groups / a.shape.heads) + in_group / wide, at = in_group % wide;
    const int2 span = a.spans[b * a.head_groups + hg];
    if (span.y <= 1) return;
    // the first part may be in either place of its workgroup, the others are in place 0 of theirs
    const size_t first = static_cast<size_t>(span.x) * wide + at, others = static_cast<size_t>(span.x / 2) * 2 * wide + at;
    auto place = [&](int i) { return i == 0 ? first : others + static_cast<size_t>(2 * wide) * i; };
    float best = -__builtin_inff();
    for (int i = lane; i < span.y; i += 64) best = fmaxf(best, a.part_ml[2 * place(i)]);
    best = across32<MaxOp>(reduce_row<MaxOp, 32>(best));
    const float from = best == -__builtin_inff() ? 0.0f : best;
    float l = 0.0f, o[EACH] = {};
    for (int base = mine; base < span.y; base += 64 * WAVES) {
        const int left = (span.y - base + WAVES - 1) / WAVES, here = left < 64 ? left : 64;
        float f = 0.0f;
        if (lane < here) {
            const size_t p = place(base + lane * WAVES);
            f = __builtin_amdgcn_exp2f(a.part_ml[2 * p] - from);
            l = __builtin_fmaf(a.part_ml[2 * p + 1], f, l);
        }
        const int weight = __builtin_bit_cast(int, f);
        for (int i = 0; i < here; i += FLIGHT) {
            part_t x[FLIGHT]; // behind the last part the last one again, which is not used
#pragma unroll
            for (int u = 0; u < FLIGHT; ++u) {
                const int j = i + u < here ? i + u : here - 1;
                x[u] = reinterpret_cast<const part_t *>(a.part_o + place(base + j * WAVES) * D)[lane];
            }
#pragma unroll
            for (int u = 0; u < FLIGHT; ++u) {
                if (i + u >= here) break;
                const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(weight, i + u));
#pragma unroll
                for (int k = 0; k < EACH; ++k) o[k] = __builtin_fmaf(x[u][k], w, o[k]);
            }
        }
    }
    l = across32<AddOp>(reduce_row<AddOp, 32>(l));
    if constexpr (WAVES > 1) {
        __shared__ float sums[WAVES][64 * EACH + 1];
#pragma unroll
        for (int k = 0; k < EACH; ++k) sums[wave][k * 64 + lane] = o[k];
        if (lane == 0) sums[wave][64 * EACH] = l;
        __syncthreads();
        if (wave > 0) return;
        l = sums[0][64 * EACH];
#pragma unroll
        for (int k = 0; k < EACH; ++k) o[k] = sums[0][k * 64 + lane];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) {
            l = l + sums[w][64 * EACH];
#pragma unroll
            for (int k = 0; k < EACH; ++k) o[k] = o[k] + sums[w][k * 64 + lane];
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t *out = reinterpret_cast<uint16_t *>(a.out) + static_cast<size_t>(row) * D + lane * EACH;
    if constexpr (EACH == 1)
        *out = static_cast<uint16_t>(pack_bf16(o[0] * inv, 0.0f));
    else if constexpr (EACH == 2)
        *reinterpret_cast<uint32_t *>(out) = pack_bf16(o[0] * inv, o[1] * inv);
    else
        *reinterpret_cast<u32x2 *>(out) = u32x2{pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv)};
    if (lane == 0 && a.lse != nullptr)
        a.lse[row] = l == 0.0f ? -__builtin_inff() : (best + __builtin_amdgcn_logf(l)) * kLn2;
}

// ------------------------------------------------------------------ the join over the ranks

template <int NSRC>
struct JoinArgs {
    const char *out[NSRC];
    const float *lse[NSRC];
    char *to;
    float *to_lse;
    size_t rows;
    int vec_shift; // log2 of the 16-byte vectors of a row
};

// out = sum_i w_i o_i / sum_i w_i, w_i = exp(lse_i - max lse): W reads and one write per element, a vector per lane
// with every source's load in flight, read once and so marked as streaming; a row whose lse is -inf is not used,
// whatever it holds.  Bound by HBM: four fp32 sources of 34 MB 31 us, 5.5 TB/s.
template <class Sum, int NSRC>
__global__ void __launch_bounds__(256)
attention_join_kernel(JoinArgs<NSRC> a)
{
    constexpr int N = kVecBytes / Sum::kElemBytes;
    const size_t items = a.rows << a.vec_shift;
    for (size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; i < items;
         i += static_cast<size_t>(gridDim.x) * 256) {
        const size_t row = i >> a.vec_shift;
        u32x4 in[NSRC];
        float w[NSRC];
#pragma unroll
        for (int s = 0; s < NSRC; ++s) in[s] = load_vec<true>(a.out[s], i);
#pragma unroll
        for (int s = 0; s < NSRC; ++s) w[s] = a.lse[s][row];
        float best = w[0];
#pragma unroll
        for (int s = 1; s < NSRC; ++s) best = fmaxf(best, w[s]);
        float total = 0.0f, o[N] = {};
#pragma unroll
        for (int s = 0; s < NSRC; ++s) {
            if (w[s] == -__builtin_inff()) continue;
            const float f = expf(w[s] - best);
            total = total + f;
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const uint32_t u = N == 4 ? in[s][k & 3] : ((k & 1) ? in[s][k >> 1] & 0xFFFF0000u : in[s][k >> 1] << 16);
                o[k] = __builtin_fmaf(bits_to_f32(u), f, o[k]);
            }
        }
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        u32x4 r;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            r[k] = N == 4 ? f32_to_bits(o[k] * inv) : pack_bf16(o[2 * k % N] * inv, o[(2 * k + 1) % N] * inv);
        store_vec<false>(a.to, i, r);
        if ((i & ((static_cast<size_t>(1) << a.vec_shift) - 1)) == 0)
            a.to_lse[row] = total == 0.0f ? -__builtin_inff() : best + logf(total);
    }
}

template <class Sum, int NSRC>
static hipError_t launch_join(const void *const *outs, const void *const *lses, void *to, float *to_lse, size_t rows,
                              int dim, hipStream_t stream)
{
    JoinArgs<NSRC> a = {};
    for (int i = 0; i < NSRC; ++i) {
        a.out[i] = static_cast<const char *>(outs[i]);
        a.lse[i] = static_cast<const float *>(lses[i]);
    }
    a.to = static_cast<char *>(to);
    a.to_lse = to_lse;
    a.rows = rows;
    a.vec_shift = __builtin_ctz(dim * Sum::kElemBytes / kVecBytes);
    const size_t need = ((rows << a.vec_shift) + 255) / 256, most = static_cast<size_t>(compute_units()) * 8;
    hipLaunchKernelGGL((attention_join_kernel<Sum, NSRC>), dim3(static_cast<unsigned>(need < most ? need : most)),
                       dim3(256), 0, stream, a);
    return hipGetLastError();
}

template <class Sum>
static hipError_t launch_join_nsrc(const void *const *outs, const void *const *lses, int world, void *to,
                                   float *to_lse, size_t rows, int dim, hipStream_t s)
{
    switch (world) {
    case 1: return launch_join<Sum, 1>(outs, lses, to, to_lse, rows, dim, s);
    case 2: return launch_join<Sum, 2>(outs, lses, to, to_lse, rows, dim, s);
    case 3: return launch_join<Sum, 3>(outs, lses, to, to_lse, rows, dim, s);
    case 4: return launch_join<Sum, 4>(outs, lses, to, to_lse, rows, dim, s);
    case 5: return launch_join<Sum, 5>(outs, lses, to, to_lse, rows, dim, s);
    case 6: return launch_join<Sum, 6>(outs, lses, to, to_lse, rows, dim, s);
    case 7: return launch_join<Sum, 7>(outs, lses, to, to_lse, rows, dim, s);
    case 8: return launch_join<Sum, 8>(outs, lses, to, to_lse, rows, dim, s);
    default: return hipErrorInvalidValue;
    }
}

// ------------------------------------------------------------------ launch shape

struct AttnPlan {
    int blocks_per_wg, head_groups, workgroups;
    size_t part_floats, span_bytes, workspace;
};

// How many workgroups share the tokens: two per compute unit (one of head_dim 256, whose registers fill it), but
// no more than there are units.  Times here and below are whole calls in a graph, lengths from a quarter of the longest
// to the longest.  64 sequences of up to 8,192 tokens, 8 key heads of 128, in 8 bits: one 128 us, two 119, three
// 130 (in bf16 207 to 208 all of them); 3 of up to 200,003 and one key head of 256: one 92, two 102.  A workgroup per row
// and no second launch instead (bf16, 8 key heads of 128)
//   - where no sequence has over 512 tokens: 32 x 500 tokens 13.5 us against 17.0 (32 x 1,000, which are shared: 25.6 against
//     21.3, so that the border could lie higher);
//   - where the rows alone fill the GPU eight times and none is so long that the last one would be waited for:
//     512 x 500 tokens 110 us against 130, 256 x 1,000 111 against 120; 128 x 2,000, whose rows do not, 113 against 115.
// Three blocks of 16 query heads and more on a key head: four waves on the same tokens, which share their loads (of three blocks
// the fourth wave loads along and multiplies zeros).  33 heads on one key head, 8 x 40,000 tokens: 37 us with four waves,
// 38 with two and so two workgroups, 55 with one and three (128 dims), 61, 68 and 92 (256), 34, 33 and 36 (128 in 8 bits);
// 64 heads 39, 39 and 65; 68, 72 and 120; 37, 36 and 43.  Short rows lose by it: 64 x 500 tokens 21, 15 and 13 us.
static AttnPlan plan_attention(size_t batch, int q_heads, int kv_heads, int head_dim, int most)
{
    AttnPlan p = {};
    const int blocks = (q_heads / kv_heads + 15) / 16;
    p.blocks_per_wg = blocks >= 3 ? 4 : blocks;
    p.head_groups = kv_heads * ((blocks + p.blocks_per_wg - 1) / p.blocks_per_wg);
    const size_t rows = batch * p.head_groups, units = compute_units();
    const size_t most_units = rows * ((static_cast<size_t>(most) + 127) / 128); // a unit is 128 or 256 tokens
    if (most <= 512 || (rows >= 8 * units && most <= 2048) || most_units >= (static_cast<size_t>(1) << 31)) return p;
    const size_t at_once = units * (head_dim == 256 ? 1 : 2), wgs = at_once < most_units ? at_once : most_units;
    p.workgroups = static_cast<int>(wgs);
    p.part_floats = 2 * wgs * 16 * p.blocks_per_wg * head_dim;
    p.span_bytes = rows * sizeof(int2);
    p.workspace = p.part_floats * sizeof(float) + p.part_floats / head_dim * 2 * sizeof(float) + p.span_bytes;
    return p;
}

// What the launches of a batch need, one after the other: all but the last have kBatch sequences.
static size_t attention_workspace(size_t batch, int q_heads, int kv_heads, int head_dim, int most)
{
    const size_t whole = batch < kBatch ? batch : kBatch, last = batch % kBatch;
    const size_t a = plan_attention(whole, q_heads, kv_heads, head_dim, most).workspace;
    const size_t b = plan_attention(last, q_heads, kv_heads, head_dim, most).workspace;
    return a > b ? a : b;
}

template <class Store, int D>
static hipError_t launch_attention(const AttnArgs &a, hipStream_t stream)
{
    const size_t grid = a.workgroups > 0 ? a.workgroups : static_cast<size_t>(a.batch) * a.head_groups;
    // what one wave alone reads is marked as streaming (64 x up to 8,192 tokens of 8 key heads in 8 bits 120 us against 136), what
    // waves share is not (3 x up to 200,003 tokens, 24 heads on one key head of 256, 91 us against 114)
    if (a.blocks_per_wg == 1)
        hipLaunchKernelGGL((decode_attention_kernel<Store, D, true>), dim3(static_cast<unsigned>(grid)),
                           dim3(kAttnBlock), 0, stream, a);
    else
        hipLaunchKernelGGL((decode_attention_kernel<Store, D, false>), dim3(static_cast<unsigned>(grid)),
                           dim3(kAttnBlock), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.workgroups == 0) return e;
    const unsigned rows = static_cast<unsigned>(a.batch) * a.q_heads;
    // four waves per row where a row has eight parts or more on average: 72 rows of 85 parts 8 us against 28 with one, while
    // 4,096 rows of two or three take 5 us with one against 11
    if (static_cast<size_t>(a.workgroups) >= 8 * static_cast<size_t>(a.batch) * a.head_groups)
        hipLaunchKernelGGL((join_parts_kernel<D, 4>), dim3(rows), dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL((join_parts_kernel<D, 1>), dim3((rows + 3) / 4), dim3(256), 0, stream, a);
    return hipGetLastError();
}

template <class Store>
static hipError_t launch_attention_dim(const AttnArgs &a, int dim, hipStream_t stream)
{
    switch (dim) {
    case 64: return launch_attention<Store, 64>(a, stream);
    case 128: return launch_attention<Store, 128>(a, stream);
    case 256: return launch_attention<Store, 256>(a, stream);
    default: return hipErrorInvalidValue;
    }
}

static int check_attention_shape(size_t batch, int q_heads, int kv_heads, int most)
{
    if (q_heads < 1 || q_heads > 65536 || kv_heads < 1 || q_heads % kv_heads != 0) return TCCL_EINVAL;
    if (most < 0 || most > (1 << 30)) return TCCL_EINVAL;
    if (batch > (static_cast<size_t>(1) << 20)) return TCCL_EINVAL;
    return TCCL_OK;
}

} // namespace tccl

using namespace tccl;

extern "C" size_t tccl_decode_attention_workspace(size_t batch, int q_heads, int kv_heads, int head_dim, int max_tokens)
{
    if (check_attention_shape(batch, q_heads, kv_heads, max_tokens) != TCCL_OK) return 0;
    return attention_workspace(batch, q_heads, kv_heads, head_dim, max_tokens);
}

extern "C" int tccl_decode_attention(const tccl_paged_cache *cache, const void *q, size_t q_batch_stride,
                                     size_t q_head_stride, const int32_t *page_table, size_t page_table_stride,
                                     const int32_t *lengths, void *out, float *lse, void *workspace,
                                     size_t workspace_bytes, size_t batch, int q_heads, int max_tokens, float scale,
                                     void *stream)
{
    AttnArgs a = {};
    if (const int rc = check_cache(cache, &a.shape)) return rc;
    if (const int rc = check_attention_shape(batch, q_heads, cache->kv_heads, max_tokens)) return rc;
    if (q == nullptr || lengths == nullptr || out == nullptr) return TCCL_EINVAL;
    if (max_tokens > 0 && page_table == nullptr) return TCCL_EINVAL;
    a.q_batch = q_batch_stride * 2;
    a.q_head = q_head_stride * 2;
    if (!aligned16(q) || !aligned16(out) || !aligned16(workspace) || (a.q_batch | a.q_head) % kVecBytes != 0)
        return TCCL_EALIGN;
    if (batch == 0) return TCCL_OK;
    const size_t need = attention_workspace(batch, q_heads, cache->kv_heads, cache->head_dim, max_tokens);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return TCCL_ESCRATCH;
    if (!fits_launch((batch < kBatch ? batch : kBatch) * q_heads, kAttnBlock)) return TCCL_EINVAL;
    a.table_row = page_table_stride;
    a.q_heads = q_heads;
    a.group = q_heads / cache->kv_heads;
    a.most = max_tokens;
    a.scale = scale * kLog2e;
    hipStream_t s = static_cast<hipStream_t>(stream);
    for (size_t first = 0; first < batch; first += kBatch) {
        const size_t here = batch - first < kBatch ? batch - first : kBatch;
        const AttnPlan plan = plan_attention(here, q_heads, cache->kv_heads, cache->head_dim, max_tokens);
        a.q = static_cast<const char *>(q) + first * a.q_batch;
        a.table = page_table + first * page_table_stride;
        a.lengths = lengths + first;
        a.out = static_cast<char *>(out) + first * q_heads * cache->head_dim * 2;
        a.lse = lse == nullptr ? nullptr : lse + first * q_heads;
        // the workspace: partial outputs, their maxima and sums, the rows' spans
        a.part_o = static_cast<float *>(workspace);
        a.part_ml = a.part_o + plan.part_floats;
        a.spans = reinterpret_cast<int2 *>(a.part_ml + plan.part_floats / cache->head_dim * 2);
        a.batch = static_cast<int>(here);
        a.blocks_per_wg = plan.blocks_per_wg;
        a.head_groups = plan.head_groups;
        a.workgroups = plan.workgroups;
        const hipError_t e = cache->dtype == TCCL_E4M3 ? launch_attention_dim<E4m3Store>(a, cache->head_dim, s)
                                                       : launch_attention_dim<Bf16Store>(a, cache->head_dim, s);
        if (e != hipSuccess) return hip_code(e);
    }
    return TCCL_OK;
}

extern "C" int tccl_attention_all_reduce(const void *const *outs, const void *const *lses, int world, void *out,
                                         float *lse, size_t rows, int head_dim, int dtype, void *stream)
{
    if (outs == nullptr || lses == nullptr || out == nullptr || lse == nullptr) return TCCL_EINVAL;
    if (world < 1 || world > TCCL_MAX_WORLD || (head_dim != 64 && head_dim != 128 && head_dim != 256))
        return TCCL_EINVAL;
    if (dtype != TCCL_BF16 && dtype != TCCL_F32) return TCCL_EINVAL;
    if (!aligned16(out) || !aligned16(lse)) return TCCL_EALIGN;
    for (int i = 0; i < world; ++i) {
        if (outs[i] == nullptr || lses[i] == nullptr) return TCCL_EINVAL;
        if (!aligned16(outs[i]) || !aligned16(lses[i])) return TCCL_EALIGN;
    }
    if (rows == 0) return TCCL_OK;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return hip_code(dtype == TCCL_BF16
                        ? launch_join_nsrc<Bf16Sum>(outs, lses, world, out, lse, rows, head_dim, s)
                        : launch_join_nsrc<F32Sum>(outs, lses, world, out, lse, rows, head_dim, s));
}

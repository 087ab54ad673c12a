// attention.hip -- attention of one new token per sequence over the paged cache of all ranks, split over the
// cache's length and joined; and the softmax-weighted all-reduce that joins the ranks' own partial
// attentions.
//
//   o = sum_t p_t v_t / sum_t p_t,  p_t = exp(s_t - m),  s_t = scale q.k_t,  m = max_t s_t,  lse = m + log sum_t p_t
// A part of the tokens gives (m, l = sum p, O = sum p v) with its own m; parts join by
//   m = max m_i,  l = sum l_i exp(m_i - m),  O = sum O_i exp(m_i - m)
// in any grouping.  No tokens give o = 0 and lse = -inf.
//
// The cache is read once; that is the floor.  A workgroup takes one sequence, one key head, up to 16 of
// the query heads that share it and one chunk of tokens, its four waves alternate blocks of tokens.  Scores
// come as S^T = K Q^T and the output as O^T = V^T P^T from 16x16x32 matrix instructions: the cache's layout makes
// every 16-byte load an operand as it stands, and a lane's scores are the tokens that the lane holds of P, so
// nothing passes through LDS and a query head's running maximum and sum stay with one lane column.
#include "host.h"
#include "rows.h"

namespace tccl {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kAttnBlock = 256;
constexpr int kAttnWaves = 4;
constexpr int kMaxChunk = 8192;  // tokens of a workgroup: 512 pages of 16
constexpr int kChunkStep = 256;  // chunks are whole pages of every size
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
    float *part_o, *part_ml; // [batch][q_heads][splits][D] and [batch][q_heads][splits][2]
    int q_heads, group, head_blocks; // query heads, per key head, and blocks of 16 of the latter
    int most, chunk, splits; // tokens: of a sequence at most, of a workgroup; chunks of `most`
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

// Lane layout, lane = 16 g + m:
//   K operand    row m is a token, the lane's 16 bytes are its dims 16-byte chunk g of four
//   Q operand    column m is a query head, the same dims
//   S^T          column m is the query head, rows 4 g + i
//   V^T operand  row m is a dim, the lane's 16 bytes are tokens of group g
//   P^T operand  column m is the query head, the same tokens
// A block is four groups of TOKENS = 8 (bf16) or 16 (8 bits) consecutive tokens.  Row 4 g + i of the block's
// K tile t is token TOKENS g + 4 t + i, so that S^T leaves the tokens of group g in lanes 16 g ... 16 g + 15,
// where P^T needs them.
template <class Store, int D>
__global__ void __launch_bounds__(kAttnBlock)
decode_attention_kernel(AttnArgs a)
{
    constexpr int TOKENS = Store::kChunk, TILES = TOKENS / 4, BLOCK = 4 * TOKENS;
    constexpr int KLOADS = D / (4 * Store::kChunk);          // 16-byte chunks of a token's row per lane
    constexpr int QSTEPS = D / 32, DTILES = D / 16, PARTS = TOKENS / 8;
    __shared__ const char *pages[kMaxChunk / 16];
    __shared__ float wave_m[kAttnWaves][16], wave_l[kAttnWaves][16];
    __shared__ float wave_o[kAttnWaves][16][D + 4];

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, m = lane & 15;
    // blockIdx.x = ((b * heads + h) * head_blocks + hb) * splits + split
    uint32_t rest = blockIdx.x;
    const int split = rest % a.splits;
    rest /= a.splits;
    const int hb = rest % a.head_blocks;
    rest /= a.head_blocks;
    const int h = rest % a.shape.heads, b = rest / a.shape.heads;
    const int length = sequence_length(a, b);
    const int begin = split * a.chunk;
    const int in_block = a.group - 16 * hb < 16 ? a.group - 16 * hb : 16; // query heads here
    const int first_head = h * a.group + 16 * hb;
    if (begin >= length && split > 0) return;
    const int end = begin + a.chunk < length ? begin + a.chunk : length;
    const int count = end - begin; // tokens; 0 only where the sequence is empty

    const int shift = a.shape.page_shift, page_size = 1 << shift;
    const int npages = (count + page_size - 1) >> shift;
    for (int i = threadIdx.x; i < npages; i += kAttnBlock)
        pages[i] = a.shape.block(a.table[static_cast<size_t>(b) * a.table_row + (begin >> shift) + i], h);

    u32x4 q[QSTEPS];
#pragma unroll
    for (int s = 0; s < QSTEPS; ++s) {
        // the dims of contraction step s that lane group g holds
        const int dim = Store::kScaled ? (s >> 1) * 64 + g * 16 + (s & 1) * 8 : s * 32 + g * 8;
        q[s] = u32x4{0, 0, 0, 0};
        if (m < in_block)
            q[s] = load_vec<false>(a.q + b * a.q_batch + (first_head + m) * a.q_head + dim * 2, 0);
    }
    __syncthreads();

    const size_t v_at = static_cast<size_t>(page_size) * D * Store::kBytes;
    const char *const safe = a.shape.pool.p[0]; // read, and masked, where there is no page
    float top = -__builtin_inff(), total = 0.0f;
    f32x4 acc[DTILES];
#pragma unroll
    for (int i = 0; i < DTILES; ++i) acc[i] = f32x4{0, 0, 0, 0};

    for (int start = wave * BLOCK; start < count; start += kAttnWaves * BLOCK) {
        // keys: lane m's token of tile t lies in group m / 4; values and scores: group g
        const int kt = start + (m >> 2) * TOKENS, vt = start + g * TOKENS;
        const int kp = kt >> shift, vp = vt >> shift;
        const char *kb = kp < npages ? pages[kp] : nullptr;
        const char *vb = vp < npages ? pages[vp] : nullptr;
        int live = vb != nullptr ? count - vt : 0; // tokens of group g that count
        live = live < 0 ? 0 : live;
        kb = kb != nullptr ? kb : safe;
        vb = vb != nullptr ? vb : safe;
        const int ko = kt & (page_size - 1), vo = vt & (page_size - 1);
        u32x4 k[TILES][KLOADS], v[DTILES];
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const int at = ko + 4 * t + (m & 3);
            const char *row = kb + static_cast<size_t>(at >> 4) * (D / Store::kChunk) * 256 + (at & 15) * 16;
#pragma unroll
            for (int c = 0; c < KLOADS; ++c) k[t][c] = load_vec<false>(row + (c * 4 + g) * 256, 0);
        }
#pragma unroll
        for (int d = 0; d < DTILES; ++d)
            v[d] = load_vec<false>(vb + v_at + (static_cast<size_t>(vo / TOKENS) * D + d * 16 + m) * 16, 0);
        float s[TILES][4], pv[TILES][4];
        u32x4 k_scales, v_scales;
        if constexpr (Store::kScaled) {
            k_scales = load_vec<false>(vb + 2 * v_at + vo, 0);
            v_scales = load_vec<false>(vb + 2 * v_at + page_size + vo, 0);
        }
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            f32x4 c = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < KLOADS; ++i) {
                if constexpr (Store::kScaled) {
                    c = mfma(widen_e4m3(k[t][i][0], k[t][i][1]), q[2 * i], c);
                    c = mfma(widen_e4m3(k[t][i][2], k[t][i][3]), q[2 * i + 1], c);
                } else {
                    c = mfma(k[t][i], q[i], c);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = c[i] * a.scale;
                if constexpr (Store::kScaled) x = x * scale_of((k_scales[t] >> (8 * i)) & 0xFFu);
                s[t][i] = 4 * t + i < live ? x : -__builtin_inff();
            }
        }
        float best = s[0][0];
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) best = fmaxf(best, s[t][i]);
        best = across32<MaxOp>(across16<MaxOp>(best));
        if (__any(best > top)) {
            const float next = fmaxf(top, best);
            const float f = next == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(top - next);
            top = next;
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
                pv[t][i] = p;
                if constexpr (Store::kScaled)
                    pv[t][i] = 4 * t + i < live ? p * scale_of((v_scales[t] >> (8 * i)) & 0xFFu) : 0.0f;
            }
        if (!__all(live >= TOKENS)) { // what lies behind the last token may be anything, NaN too
#pragma unroll
            for (int d = 0; d < DTILES; ++d)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    constexpr int EACH = 4 / Store::kBytes;
                    const int in_word = live - w * EACH;
                    const uint32_t keep = in_word >= EACH ? ~0u : (in_word <= 0 ? 0u : (1u << (8 * Store::kBytes * in_word)) - 1u);
                    v[d][w] &= keep;
                }
        }
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            // P in two bf16 terms, so that its rounding (2^-9 of each weight) does not reach the output
            u32x4 hi, lo;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float x = pv[2 * part + (w >> 1)][(2 * w) & 3], y = pv[2 * part + (w >> 1)][(2 * w + 1) & 3];
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
    }

    // the four waves' parts: lane groups hold the sums of their own tokens, and all dims of O
    total = across32<AddOp>(across16<AddOp>(total));
    if (g == 0) {
        wave_m[wave][m] = top;
        wave_l[wave][m] = total;
    }
#pragma unroll
    for (int d = 0; d < DTILES; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) wave_o[wave][m][d * 16 + 4 * g + i] = acc[d][i];
    __syncthreads();
    const bool whole = a.splits == 1;
    for (int item = threadIdx.x; item < in_block * (D / 4); item += kAttnBlock) {
        const int n = item / (D / 4), d = item % (D / 4) * 4;
        float best = wave_m[0][n];
#pragma unroll
        for (int w = 1; w < kAttnWaves; ++w) best = fmaxf(best, wave_m[w][n]);
        const float from = best == -__builtin_inff() ? 0.0f : best;
        float l = 0.0f;
        f32x4 o = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kAttnWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(wave_m[w][n] - from);
            l = __builtin_fmaf(wave_l[w][n], f, l);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = __builtin_fmaf(wave_o[w][n][d + i], f, o[i]);
        }
        const size_t row = static_cast<size_t>(b) * a.q_heads + first_head + n;
        if (whole) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            *reinterpret_cast<u32x2 *>(a.out + (row * D + d) * 2) =
                u32x2{pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv)};
            if (d == 0 && a.lse != nullptr)
                a.lse[row] = l == 0.0f ? -__builtin_inff() : (best + __builtin_amdgcn_logf(l)) * kLn2;
        } else {
            const size_t at = row * a.splits + split;
            *reinterpret_cast<f32x4 *>(a.part_o + at * D + d) = o;
            if (d == 0) {
                a.part_ml[2 * at] = best;
                a.part_ml[2 * at + 1] = l;
            }
        }
    }
}

// One workgroup per (sequence, query head): D / 4 lanes of four dims, the others take every n-th chunk.
template <int D>
__global__ void __launch_bounds__(256)
join_chunks_kernel(AttnArgs a)
{
    constexpr int LANES = D / 4, ROWS = 256 / LANES;
    __shared__ float part[ROWS][D + 2];
    const size_t row = blockIdx.x;
    const int length = sequence_length(a, static_cast<int>(row / a.q_heads));
    const int live = length == 0 ? 1 : (length + a.chunk - 1) / a.chunk;
    const int d = threadIdx.x % LANES * 4, r = threadIdx.x / LANES;
    const float *const ml = a.part_ml + row * a.splits * 2;
    const float *const po = a.part_o + row * a.splits * D;
    float best = -__builtin_inff();
    for (int i = r; i < live; i += ROWS) best = fmaxf(best, ml[2 * i]);
    if (d == 0) part[r][0] = best;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ROWS; ++i) best = fmaxf(best, part[i][0]);
    __syncthreads();
    const float from = best == -__builtin_inff() ? 0.0f : best;
    float l = 0.0f;
    f32x4 o = {0, 0, 0, 0};
    for (int i = r; i < live; i += ROWS) {
        const float f = __builtin_amdgcn_exp2f(ml[2 * i] - from);
        const f32x4 x = *reinterpret_cast<const f32x4 *>(po + static_cast<size_t>(i) * D + d);
        l = __builtin_fmaf(ml[2 * i + 1], f, l);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = __builtin_fmaf(x[k], f, o[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) part[r][d + k] = o[k];
    if (d == 0) part[r][D] = l;
    __syncthreads();
    if (r > 0) return;
    l = 0.0f;
    o = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        l = l + part[i][D];
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = o[k] + part[i][d + k];
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    *reinterpret_cast<u32x2 *>(a.out + (row * D + d) * 2) =
        u32x2{pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv)};
    if (d == 0 && a.lse != nullptr)
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
    int lane_shift; // log2 of the lanes of a row
};

// out = sum_i w_i o_i / sum_i w_i, w_i = exp(lse_i - max lse): W reads and one write per element, so a
// grid-stride pass with every source's load in flight; a row whose lse is -inf is not used, whatever it holds.
template <class Row, int NSRC>
__global__ void __launch_bounds__(256)
attention_join_kernel(JoinArgs<NSRC> a)
{
    const size_t items = a.rows << a.lane_shift;
    for (size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; i < items;
         i += static_cast<size_t>(gridDim.x) * 256) {
        const size_t row = i >> a.lane_shift;
        Row in[NSRC];
        float w[NSRC];
#pragma unroll
        for (int s = 0; s < NSRC; ++s) w[s] = a.lse[s][row];
#pragma unroll
        for (int s = 0; s < NSRC; ++s) in[s].load(a.out[s] + i * 8 * Row::kElemBytes);
        float best = w[0];
#pragma unroll
        for (int s = 1; s < NSRC; ++s) best = fmaxf(best, w[s]);
        float total = 0.0f, o[8] = {};
#pragma unroll
        for (int s = 0; s < NSRC; ++s) {
            if (w[s] == -__builtin_inff()) continue;
            const float f = expf(w[s] - best);
            total = total + f;
#pragma unroll
            for (int k = 0; k < 8; ++k) o[k] = __builtin_fmaf(in[s].at(k), f, o[k]);
        }
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = o[k] * inv;
        Row::store(a.to + i * 8 * Row::kElemBytes, o);
        if ((i & ((static_cast<size_t>(1) << a.lane_shift) - 1)) == 0)
            a.to_lse[row] = total == 0.0f ? -__builtin_inff() : best + logf(total);
    }
}

template <class Row, int NSRC>
static hipError_t launch_join(const void *const *outs, const void *const *lses, void *to, float *to_lse, size_t rows,
                              int lane_shift, hipStream_t stream)
{
    JoinArgs<NSRC> a = {};
    for (int i = 0; i < NSRC; ++i) {
        a.out[i] = static_cast<const char *>(outs[i]);
        a.lse[i] = static_cast<const float *>(lses[i]);
    }
    a.to = static_cast<char *>(to);
    a.to_lse = to_lse;
    a.rows = rows;
    a.lane_shift = lane_shift;
    const size_t need = ((rows << lane_shift) + 255) / 256, most = static_cast<size_t>(compute_units()) * 8;
    hipLaunchKernelGGL((attention_join_kernel<Row, NSRC>), dim3(static_cast<unsigned>(need < most ? need : most)),
                       dim3(256), 0, stream, a);
    return hipGetLastError();
}

template <class Row>
static hipError_t launch_join_nsrc(const void *const *outs, const void *const *lses, int world, void *to,
                                   float *to_lse, size_t rows, int lane_shift, hipStream_t s)
{
    switch (world) {
    case 1: return launch_join<Row, 1>(outs, lses, to, to_lse, rows, lane_shift, s);
    case 2: return launch_join<Row, 2>(outs, lses, to, to_lse, rows, lane_shift, s);
    case 3: return launch_join<Row, 3>(outs, lses, to, to_lse, rows, lane_shift, s);
    case 4: return launch_join<Row, 4>(outs, lses, to, to_lse, rows, lane_shift, s);
    case 5: return launch_join<Row, 5>(outs, lses, to, to_lse, rows, lane_shift, s);
    case 6: return launch_join<Row, 6>(outs, lses, to, to_lse, rows, lane_shift, s);
    case 7: return launch_join<Row, 7>(outs, lses, to, to_lse, rows, lane_shift, s);
    case 8: return launch_join<Row, 8>(outs, lses, to, to_lse, rows, lane_shift, s);
    default: return hipErrorInvalidValue;
    }
}

// ------------------------------------------------------------------ launch shape

struct AttnPlan {
    int chunk, splits, head_blocks;
    size_t workspace;
};

// Chunks such that the launch has about four workgroups per compute unit if every sequence has `most` tokens,
// in steps of 256 tokens.
static AttnPlan plan_attention(size_t batch, int q_heads, int kv_heads, int head_dim, int most)
{
    AttnPlan p;
    p.head_blocks = (q_heads / kv_heads + 15) / 16;
    const size_t rows = batch * kv_heads * p.head_blocks;
    const size_t want = static_cast<size_t>(compute_units()) * 4;
    size_t splits = rows == 0 ? 1 : (want + rows - 1) / rows;
    size_t chunk = (static_cast<size_t>(most) + splits - 1) / splits;
    chunk = (chunk + kChunkStep - 1) / kChunkStep * kChunkStep;
    chunk = chunk < kChunkStep ? kChunkStep : (chunk > kMaxChunk ? kMaxChunk : chunk);
    p.chunk = static_cast<int>(chunk);
    p.splits = most <= 0 ? 1 : static_cast<int>((static_cast<size_t>(most) + chunk - 1) / chunk);
    p.workspace = p.splits == 1 ? 0 : batch * q_heads * p.splits * (head_dim + 2) * sizeof(float);
    return p;
}

template <class Store, int D>
static hipError_t launch_attention(const AttnArgs &a, size_t batch, hipStream_t stream)
{
    const size_t grid = batch * a.shape.heads * a.head_blocks * a.splits;
    hipLaunchKernelGGL((decode_attention_kernel<Store, D>), dim3(static_cast<unsigned>(grid)), dim3(kAttnBlock), 0,
                       stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.splits == 1) return e;
    hipLaunchKernelGGL((join_chunks_kernel<D>), dim3(static_cast<unsigned>(batch * a.q_heads)), dim3(256), 0, stream,
                       a);
    return hipGetLastError();
}

template <class Store>
static hipError_t launch_attention_dim(const AttnArgs &a, size_t batch, int dim, hipStream_t stream)
{
    switch (dim) {
    case 64: return launch_attention<Store, 64>(a, batch, stream);
    case 128: return launch_attention<Store, 128>(a, batch, stream);
    case 256: return launch_attention<Store, 256>(a, batch, stream);
    default: return hipErrorInvalidValue;
    }
}

static int check_attention_shape(size_t batch, int q_heads, int kv_heads, int most)
{
    if (q_heads < 1 || q_heads > 65536 || kv_heads < 1 || q_heads % kv_heads != 0 || most < 0) return TCCL_EINVAL;
    if (batch > (static_cast<size_t>(1) << 20)) return TCCL_EINVAL;
    return TCCL_OK;
}

} // namespace tccl

using namespace tccl;

extern "C" size_t tccl_decode_attention_workspace(size_t batch, int q_heads, int kv_heads, int head_dim, int max_tokens)
{
    if (check_attention_shape(batch, q_heads, kv_heads, max_tokens) != TCCL_OK) return 0;
    return plan_attention(batch, q_heads, kv_heads, head_dim, max_tokens).workspace;
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
    const AttnPlan plan = plan_attention(batch, q_heads, cache->kv_heads, cache->head_dim, max_tokens);
    if (plan.workspace > 0 && (workspace == nullptr || workspace_bytes < plan.workspace)) return TCCL_ESCRATCH;
    if (batch * cache->kv_heads * plan.head_blocks * plan.splits > 0x7FFFFFFFull || batch * q_heads > 0x7FFFFFFFull)
        return TCCL_EINVAL;
    a.q = static_cast<const char *>(q);
    a.table = page_table;
    a.table_row = page_table_stride;
    a.lengths = lengths;
    a.out = static_cast<char *>(out);
    a.lse = lse;
    // the maxima and sums lie behind the partial outputs
    a.part_o = static_cast<float *>(workspace);
    a.part_ml = a.part_o + (plan.workspace > 0 ? batch * q_heads * plan.splits * cache->head_dim : 0);
    a.q_heads = q_heads;
    a.group = q_heads / cache->kv_heads;
    a.head_blocks = plan.head_blocks;
    a.most = max_tokens;
    a.chunk = plan.chunk;
    a.splits = plan.splits;
    a.scale = scale * kLog2e;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return hip_code(cache->dtype == TCCL_E4M3 ? launch_attention_dim<E4m3Store>(a, batch, cache->head_dim, s)
                                              : launch_attention_dim<Bf16Store>(a, batch, cache->head_dim, s));
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
    const int shift = head_dim == 64 ? 3 : (head_dim == 128 ? 4 : 5);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return hip_code(dtype == TCCL_BF16
                        ? launch_join_nsrc<Bf16Row>(outs, lses, world, out, lse, rows, shift, s)
                        : launch_join_nsrc<F32Row>(outs, lses, world, out, lse, rows, shift, s));
}

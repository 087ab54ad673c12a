// qk_norm.hip -- a one-shot all-reduce of the ranks' partial query/key/value projections whose epilogue
// norms every query and key head and rotates it by its token's position, and its backward pass.
//
//   x = sum_i buf_i            fp32, rank order; a head is head_dim consecutive elements
//   r = 1 / sqrt(mean x^2 + eps),  n = x r,  h = n w          (q_weight for query heads, k_weight for key heads)
//   y = R(position) h          pairs (a, b) -> (a cos - b sin, b cos + a sin), angle position * inv_freq[i]
// value heads behind the keys are only summed.  Backward, with g = R^T dy, u = g w:
//   dx = r (u - n mean(u n)),  dw = sum over tokens and heads of g n
//
// Memory-bound: W reads and one write per element, a few dozen operations each.  A lane holds eight
// elements, so a wave works on 512 consecutive elements (four heads of 128) with one 16-byte load per
// source; the mean is a reduction over head_dim / 8 lanes in registers.  Angles are formed in fp64 turns
// (fp32 would lose the fraction of a far position's angle) once per token by the workgroup, into LDS.
// Measured: forward, 4,099 tokens of 48 heads of 128, 8 bf16 sources 78 us, 5.8 TB/s; 8,191 tokens of 20 heads of 256, one
// fp32 source 63 us, 5.3 TB/s read and written; backward, 8,192 tokens of 48 heads of 128, one bf16 source 52 to 53 us, 5.4 TB/s;
// 777 tokens of 36 heads of 64, four fp32 sources 11.8 us, 2.9 TB/s: five items for four waves, one of which works twice.
#include <type_traits>

#include "host.h"
#include "rows.h"

namespace tccl {

constexpr int kNormBlock = 256;
constexpr int kNormWaves = kNormBlock / 64;
constexpr int kNormTokens = 4; // most tokens a workgroup works on at once
constexpr int kMaxRotary = 256;

template <int NSRC>
struct NormArgs {
    const char *src[NSRC];
    char *out[3];        // forward: q, k, v;  backward: dx, unused, unused
    const char *grad[3]; // backward: dq, dk, dv
    const char *weight[2];
    const int64_t *positions;
    const double *inv_freq;
    float *partial; // backward: [workgroups][2][head_dim] sums of g n
    size_t tokens;
    int heads[3];
    int rotary, interleaved;
    int tokens_per_wg; // 1, 2 or 4
    float eps;
};

// cos and sin of position * inv_freq[i].  The angle is reduced to (-1/2, 1/2] turns in fp64.
__device__ __forceinline__ f32x2 rotation(int64_t position, double inv_freq)
{
    double turns = static_cast<double>(position) * inv_freq * 0.15915494309189533577;
    turns = turns - __builtin_rint(turns);
    const float half_turns = static_cast<float>(turns + turns);
    return f32x2{cospif(half_turns), sinpif(half_turns)};
}

// The workgroup's (cos, sin) pairs, [token][rotary / 2], and kTurns behind them (cos, -sin).  A lane needs `each` = 8
// pairs that follow each other (4 where neighbours are pairs); two of them are one 16-byte read, and these lie
// lane by lane, so that a row's reads, and those of the lanes that take the other sign, fall into different banks.
constexpr int kTurns = kNormTokens * kMaxRotary / 2 + 16;
__device__ __forceinline__ int turn_place(int pair, int each, int lanes)
{
    const int lane = pair / each, k = pair % each;
    return ((k >> 1) * lanes + lane) * 2 + (k & 1);
}

// A lane's eight elements, rotated (SIGN = 1) or rotated back (-1); `place` is the lane's place in its row.
template <int LANES, int SIGN>
__device__ __forceinline__ void rotate(float *x, const f32x2 *turn, int place, int rotary, bool interleaved)
{
    const int lanes = rotary >> 3;
    if (interleaved) {
        if (place < lanes) {
            const f32x2 *t = turn + (SIGN < 0 ? kTurns : 0) + 2 * place;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const f32x2 cs = t[(k >> 1) * 2 * lanes + (k & 1)];
                const float u = x[2 * k], v = x[2 * k + 1];
                x[2 * k] = __builtin_fmaf(u, cs.x, -(v * cs.y));
                x[2 * k + 1] = __builtin_fmaf(v, cs.x, u * cs.y);
            }
        }
    } else {
        const int half = lanes >> 1;
        const bool low = place < half;
        float y[8]; // the other half's
        if (LANES == 16 && lanes == LANES) {
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = dpp<kDppRotate8>(x[k]);
        } else {
            const int lane = threadIdx.x & 63;
            const int from = (lane & ~(LANES - 1)) + (place >= lanes ? place : (low ? place + half : place - half));
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = __shfl(x[k], from);
        }
        if (place < lanes) {
            const f32x2 *t = turn + (low == (SIGN > 0) ? kTurns : 0) + 2 * (low ? place : place - half);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const f32x2 cs = t[(k >> 1) * 2 * half + (k & 1)];
                x[k] = __builtin_fmaf(x[k], cs.x, y[k] * cs.y);
            }
        }
    }
}

template <class Row, int NSRC>
__device__ __forceinline__ void sum_sources(const Row *in, float *x)
{
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        float a = 0.0f;
#pragma unroll
        for (int i = 0; i < NSRC; ++i) a = a + in[i].at(k);
        x[k] = a;
    }
}

template <int LANES>
__device__ __forceinline__ float inverse_rms(const float *x, float eps)
{
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s = __builtin_fmaf(x[k], x[k], s);
    return rsqrtf(__builtin_fmaf(reduce_row<AddOp, LANES>(s), 1.0f / (8 * LANES), eps));
}

// The angles of the workgroup's tokens.  A place behind the last token is no rotation (and not what LDS happens to
// hold: a missing token's zeros have to stay zeros).
template <int NSRC>
__device__ __forceinline__ void fill_angles(const NormArgs<NSRC> &a, f32x2 *turn, size_t first)
{
    const int half = a.rotary >> 1;
    for (int i = threadIdx.x; i < half * a.tokens_per_wg; i += kNormBlock) {
        const size_t t = first + i / half;
        const f32x2 cs = t < a.tokens ? rotation(a.positions[t], a.inv_freq[i % half]) : f32x2{1.0f, 0.0f};
        const int each = a.interleaved ? 4 : 8, to = i / half * half + turn_place(i % half, each, half / each);
        turn[to] = cs;
        turn[kTurns + to] = f32x2{cs.x, -cs.y};
    }
}

// What the heads of an item are: of one kind, which the whole wave then works on without asking, or mixed.
enum Kind { kQuery, kKey, kValue, kMixed };
template <int NSRC>
__device__ __forceinline__ Kind kind_of(const NormArgs<NSRC> &a, int head0, int heads)
{
    const int q = a.heads[0], qk = a.heads[0] + a.heads[1], all = qk + a.heads[2];
    const int last = (head0 + heads < all ? head0 + heads : all) - 1;
    return last < q ? kQuery : (head0 >= qk ? kValue : (head0 >= q && last < qk ? kKey : kMixed));
}

// A wave reads up to three items (a token's heads, 512 elements at a time) before it works on the first: 8 sources of
// 50 MB 81 us with one at a time, 80 two, 78 three, 81 four; one fp32 source of 168 MB 66, 66, 62, 62.
constexpr int kNormItems = 3;

template <class Row, int LANES, int NSRC>
__global__ void __launch_bounds__(kNormBlock)
qk_norm_rope_kernel(NormArgs<NSRC> a)
{
    constexpr int D = 8 * LANES, HEADS = 64 / LANES, BYTES = Row::kElemBytes; // heads a wave holds
    __shared__ __attribute__((aligned(16))) f32x2 turn[2 * kTurns];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), place = lane & (LANES - 1);
    const uint32_t mine_at = lane * 8 * BYTES; // heads follow each other: the lane's elements of an item
    const int all = a.heads[0] + a.heads[1] + a.heads[2];
    const int groups = (all + HEADS - 1) / HEADS, items = groups * a.tokens_per_wg;
    const size_t first = static_cast<size_t>(blockIdx.x) * a.tokens_per_wg;
    float wq[8], wk[8];
    load_row<Row>(a.weight[0] + place * 8 * BYTES, wq);
    load_row<Row>(a.weight[1] + place * 8 * BYTES, wk);
    fill_angles(a, turn, first);
    __syncthreads();
    for (int item0 = wave; item0 < items; item0 += kNormWaves * kNormItems) {
        float xs[kNormItems][8];
#pragma unroll
        for (int u = 0; u < kNormItems; ++u) {
            const int item = item0 + u * kNormWaves;
            const int local = item / groups, head0 = (item - local * groups) * HEADS;
            const size_t token = first + local, at = (token * all + head0) * D * BYTES;
            const bool live = item < items && token < a.tokens && head0 + lane / LANES < all;
            Row in[NSRC];
#pragma unroll
            for (int i = 0; i < NSRC; ++i) {
                if (live)
                    in[i].template load<true>(a.src[i] + at + mine_at);
                else
                    in[i].zero();
            }
            sum_sources<Row, NSRC>(in, xs[u]);
        }
#pragma unroll
        for (int u = 0; u < kNormItems; ++u) {
            const int item = item0 + u * kNormWaves;
            if (item >= items) break;
            const int local = item / groups, head0 = (item - local * groups) * HEADS, head = head0 + lane / LANES;
            const size_t token = first + local;
            const bool live = token < a.tokens && head < all;
            float *x = xs[u];
            auto work = [&](auto kind) {
                constexpr Kind KIND = decltype(kind)::value;
                const bool is_q = KIND == kQuery || (KIND == kMixed && head < a.heads[0]);
                const bool is_v = KIND == kValue || (KIND == kMixed && head >= a.heads[0] + a.heads[1]);
                if constexpr (KIND != kValue) {
                    const float r = inverse_rms<LANES>(x, a.eps);
                    float y[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) y[k] = x[k] * r * (is_q ? wq[k] : wk[k]);
                    rotate<LANES, 1>(y, turn + local * (a.rotary >> 1), place, a.rotary, a.interleaved != 0);
#pragma unroll
                    for (int k = 0; k < 8; ++k) x[k] = is_v ? x[k] : y[k];
                }
                const int before = is_q ? 0 : (is_v ? a.heads[0] + a.heads[1] : a.heads[0]);
                const int mine = is_q ? a.heads[0] : (is_v ? a.heads[2] : a.heads[1]);
                char *const out = is_q ? a.out[0] : (is_v ? a.out[2] : a.out[1]);
                if (live) Row::store(out + (token * mine + (head0 - before)) * D * BYTES + mine_at, x);
            };
            switch (kind_of(a, head0, HEADS)) {
            case kQuery: work(std::integral_constant<Kind, kQuery>()); break;
            case kKey: work(std::integral_constant<Kind, kKey>()); break;
            case kValue: work(std::integral_constant<Kind, kValue>()); break;
            default: work(std::integral_constant<Kind, kMixed>()); break;
            }
        }
    }
}

// Workgroups walk the tokens with the grid's stride; each lane keeps the weight gradients of its eight dims
// in registers until the end, so that a workgroup leaves one partial row and the result does not depend on
// the order in which workgroups finish.
// Workgroups that run at once on a compute unit: as many as the registers allow (8,192 tokens of 48 heads of 128, one
// bf16 source: 51 us with five, 57 with four; six spill).
constexpr int kMostGradPerUnit = 5;
template <class Row, int NSRC>
constexpr int kGradPerUnit = (Row::kElemBytes == 2 ? 5 : 4) - (NSRC > 6 ? 1 : 0);

template <class Row, int LANES, int NSRC>
__global__ void __launch_bounds__(kNormBlock, (kGradPerUnit<Row, NSRC>))
qk_norm_rope_backward_kernel(NormArgs<NSRC> a)
{
    constexpr int D = 8 * LANES, HEADS = 64 / LANES, BYTES = Row::kElemBytes;
    __shared__ __attribute__((aligned(16))) f32x2 turn[2 * kTurns];
    __shared__ float sums[kNormWaves][2][D];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), place = lane & (LANES - 1);
    const uint32_t mine_at = lane * 8 * BYTES; // heads follow each other: the lane's elements of an item
    const int all = a.heads[0] + a.heads[1] + a.heads[2];
    const int groups = (all + HEADS - 1) / HEADS, items = groups * a.tokens_per_wg;
    Row wq, wk;
    wq.load(a.weight[0] + place * 8 * BYTES);
    wk.load(a.weight[1] + place * 8 * BYTES);
    float dw[2][8] = {};
    for (size_t first = static_cast<size_t>(blockIdx.x) * a.tokens_per_wg; first < a.tokens;
         first += static_cast<size_t>(gridDim.x) * a.tokens_per_wg) {
        fill_angles(a, turn, first);
        __syncthreads();
        for (int item = wave; item < items; item += kNormWaves) {
            const int local = item / groups, head0 = (item - local * groups) * HEADS, head = head0 + lane / LANES;
            const size_t token = first + local, at = (token * all + head0) * D * BYTES;
            const bool live = token < a.tokens && head < all;
            auto work = [&](auto kind) {
                constexpr Kind KIND = decltype(kind)::value;
                const bool is_q = KIND == kQuery || (KIND == kMixed && head < a.heads[0]);
                const bool is_v = KIND == kValue || (KIND == kMixed && head >= a.heads[0] + a.heads[1]);
                const int before = is_q ? 0 : (is_v ? a.heads[0] + a.heads[1] : a.heads[0]);
                const int mine = is_q ? a.heads[0] : (is_v ? a.heads[2] : a.heads[1]);
                const char *const from = is_q ? a.grad[0] : (is_v ? a.grad[2] : a.grad[1]);
                Row in[NSRC], dy;
#pragma unroll
                for (int i = 0; i < NSRC; ++i) {
                    if (KIND != kValue && live && !is_v)
                        in[i].template load<true>(a.src[i] + at + mine_at);
                    else
                        in[i].zero();
                }
                if (live)
                    dy.template load<true>(from + (token * mine + (head0 - before)) * D * BYTES + mine_at);
                else
                    dy.zero();
                float g[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) g[k] = dy.at(k);
                auto weight = [&](int k) {
                    if constexpr (KIND == kQuery) return wq.at(k);
                    if constexpr (KIND == kKey) return wk.at(k);
                    const float q = wq.at(k), k_ = wk.at(k);
                    return is_q ? q : k_;
                };
                if constexpr (KIND != kValue) {
                    float n[8], dot = 0.0f;
                    sum_sources<Row, NSRC>(in, n);
                    // a lane without a head or token, or with a value head, holds zeros: where eps is 0 their root's inverse is
                    // infinite and 0 times it NaN, so that n is made 0 by r and adds nothing to dw
                    const float root = inverse_rms<LANES>(n, a.eps), r = live && !is_v ? root : 0.0f;
                    rotate<LANES, -1>(g, turn + local * (a.rotary >> 1), place, a.rotary, a.interleaved != 0);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        n[k] = n[k] * r;
                        const float gn = g[k] * n[k];
                        g[k] = g[k] * weight(k);
                        dot = __builtin_fmaf(g[k], n[k], dot);
                        if constexpr (KIND == kMixed) {
                            dw[0][k] = dw[0][k] + (is_q ? gn : 0.0f);
                            dw[1][k] = dw[1][k] + (is_q || is_v ? 0.0f : gn);
                        } else {
                            dw[KIND == kQuery ? 0 : 1][k] = dw[KIND == kQuery ? 0 : 1][k] + gn;
                        }
                    }
                    dot = reduce_row<AddOp, LANES>(dot) * (1.0f / D);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float d = r * __builtin_fmaf(-n[k], dot, g[k]);
                        g[k] = KIND == kMixed && is_v ? dy.at(k) : d;
                    }
                }
                if (live) Row::store(a.out[0] + at + mine_at, g);
            };
            switch (kind_of(a, head0, HEADS)) {
            case kQuery: work(std::integral_constant<Kind, kQuery>()); break;
            case kKey: work(std::integral_constant<Kind, kKey>()); break;
            case kValue: work(std::integral_constant<Kind, kValue>()); break;
            default: work(std::integral_constant<Kind, kMixed>()); break;
            }
        }
        __syncthreads();
    }
    // over the wave's heads (lanes LANES apart), then over the waves
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float s = dw[kind][k];
#pragma unroll
            for (int step = LANES; step < 64; step *= 2) s = s + __shfl_xor(s, step);
            if (lane < LANES) sums[wave][kind][place * 8 + k] = s;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += kNormBlock) {
        float s = 0.0f;
#pragma unroll
        for (int v = 0; v < kNormWaves; ++v) s = s + (&sums[v][0][0])[i];
        a.partial[static_cast<size_t>(blockIdx.x) * 2 * D + i] = s;
    }
}

// The partial rows in a fixed order: 16 columns per workgroup, every 64th row per lane with its loads in
// flight, joined through LDS.
constexpr int kGradRows = 64;
__global__ void __launch_bounds__(16 * kGradRows)
weight_grad_kernel(const float *partial, int rows, int dim, float *dq_weight, float *dk_weight)
{
    __shared__ float part[kGradRows][17];
    const int column = blockIdx.x * 16 + (threadIdx.x & 15), lane = threadIdx.x >> 4;
    float s = 0.0f;
#pragma unroll 16
    for (int r = lane; r < rows; r += kGradRows) s = s + partial[static_cast<size_t>(r) * 2 * dim + column];
    part[lane][threadIdx.x & 15] = s;
    __syncthreads();
    if (lane >= 4) return;
    for (int r = lane + 4; r < kGradRows; r += 4) s = s + part[r][threadIdx.x & 15];
    s = s + __shfl_xor(s, 16);
    s = s + __shfl_xor(s, 32);
    if (lane > 0) return;
    if (column < dim)
        dq_weight[column] = s;
    else
        dk_weight[column - dim] = s;
}

struct NormCall {
    const void *const *bufs;
    int world;
    void *out[3];
    const void *grad[3];
    const void *weight[2];
    const int64_t *positions;
    const double *inv_freq;
    float *partial;
    size_t tokens;
    int heads[3];
    int dim, rotary, interleaved;
    float eps;
    bool backward;
    unsigned workgroups;
    int tokens_per_wg;
};

template <class Row, int LANES, int NSRC>
static hipError_t launch_norm(NormCall &c, hipStream_t stream)
{
    NormArgs<NSRC> a = {};
    for (int i = 0; i < NSRC; ++i) a.src[i] = static_cast<const char *>(c.bufs[i]);
    for (int i = 0; i < 3; ++i) {
        a.out[i] = static_cast<char *>(c.out[i]);
        a.grad[i] = static_cast<const char *>(c.grad[i]);
        a.heads[i] = c.heads[i];
    }
    for (int i = 0; i < 2; ++i) a.weight[i] = static_cast<const char *>(c.weight[i]);
    a.positions = c.positions;
    a.inv_freq = c.inv_freq;
    a.partial = c.partial;
    a.tokens = c.tokens;
    a.rotary = c.rotary;
    a.interleaved = c.interleaved;
    a.tokens_per_wg = c.tokens_per_wg;
    a.eps = c.eps;
    if (c.backward) { // a partial row from each workgroup
        const unsigned most = static_cast<unsigned>(compute_units()) * kGradPerUnit<Row, NSRC>;
        c.workgroups = c.workgroups < most ? c.workgroups : most;
        hipLaunchKernelGGL((qk_norm_rope_backward_kernel<Row, LANES, NSRC>), dim3(c.workgroups), dim3(kNormBlock), 0,
                           stream, a);
    } else
        hipLaunchKernelGGL((qk_norm_rope_kernel<Row, LANES, NSRC>), dim3(c.workgroups), dim3(kNormBlock), 0, stream,
                           a);
    return hipGetLastError();
}

template <class Row, int LANES>
static hipError_t launch_norm_nsrc(NormCall &c, hipStream_t stream)
{
    switch (c.world) {
    case 1: return launch_norm<Row, LANES, 1>(c, stream);
    case 2: return launch_norm<Row, LANES, 2>(c, stream);
    case 3: return launch_norm<Row, LANES, 3>(c, stream);
    case 4: return launch_norm<Row, LANES, 4>(c, stream);
    case 5: return launch_norm<Row, LANES, 5>(c, stream);
    case 6: return launch_norm<Row, LANES, 6>(c, stream);
    case 7: return launch_norm<Row, LANES, 7>(c, stream);
    case 8: return launch_norm<Row, LANES, 8>(c, stream);
    default: return hipErrorInvalidValue;
    }
}

template <class Row>
static hipError_t launch_norm_dim(NormCall &c, hipStream_t stream)
{
    switch (c.dim) {
    case 64: return launch_norm_nsrc<Row, 8>(c, stream);
    case 128: return launch_norm_nsrc<Row, 16>(c, stream);
    case 256: return launch_norm_nsrc<Row, 32>(c, stream);
    default: return hipErrorInvalidValue;
    }
}

// Tokens a workgroup takes at once: where a token has fewer than four waves' worth of heads, more tokens.  8,192 tokens
// of three heads of 64, forward and backward: 8.7 and 11.7 us with four, 13.2 and 19.0 with one; of six heads of 128
// 15.6 and 17.0 with two, 19.6 and 22.6 with one.
static int norm_tokens_per_wg(const NormCall &c)
{
    const int per_wave = 512 / c.dim;
    const int groups = (c.heads[0] + c.heads[1] + c.heads[2] + per_wave - 1) / per_wave;
    return groups >= kNormWaves ? 1 : (groups >= 2 ? 2 : 4);
}

static unsigned norm_workgroups(const NormCall &c)
{
    return static_cast<unsigned>((c.tokens + c.tokens_per_wg - 1) / c.tokens_per_wg);
}

static int check_norm(const NormCall &c, int dtype)
{
    if (c.bufs == nullptr || c.world < 1 || c.world > TCCL_MAX_WORLD) return TCCL_EINVAL;
    if (dtype != TCCL_BF16 && dtype != TCCL_F32) return TCCL_EINVAL;
    if (c.dim != 64 && c.dim != 128 && c.dim != 256) return TCCL_EINVAL;
    if (c.heads[0] < 0 || c.heads[1] < 0 || c.heads[2] < 0) return TCCL_EINVAL;
    const int64_t all = static_cast<int64_t>(c.heads[0]) + c.heads[1] + c.heads[2];
    if (all < 1 || all > (1 << 20)) return TCCL_EINVAL;
    if (c.rotary < 0 || c.rotary > c.dim || c.rotary % 16 != 0) return TCCL_EINVAL;
    if (!(c.eps >= 0.0f)) return TCCL_EINVAL;
    if (c.weight[0] == nullptr || c.weight[1] == nullptr || c.positions == nullptr) return TCCL_EINVAL;
    if (c.rotary > 0 && c.inv_freq == nullptr) return TCCL_EINVAL;
    if (!c.backward && !fits_launch(c.tokens, kNormBlock)) return TCCL_EINVAL; // one workgroup per token at most
    if (c.tokens > 0x7FFFFFFFull) return TCCL_EINVAL;
    if (!aligned16(c.weight[0]) || !aligned16(c.weight[1])) return TCCL_EALIGN;
    for (int i = 0; i < c.world; ++i) {
        if (c.bufs[i] == nullptr) return TCCL_EINVAL;
        if (!aligned16(c.bufs[i])) return TCCL_EALIGN;
    }
    for (int i = 0; i < 3; ++i) {
        if (c.heads[i] > 0 && ((c.backward ? c.grad[i] : c.out[i]) == nullptr)) return TCCL_EINVAL;
        if (!aligned16(c.grad[i]) || !aligned16(c.out[i])) return TCCL_EALIGN;
    }
    return TCCL_OK;
}

} // namespace tccl

using namespace tccl;

extern "C" int tccl_qk_norm_rope(const void *const *bufs, int world, void *q_out, void *k_out, void *v_out,
                                 const void *q_weight, const void *k_weight, const int64_t *positions,
                                 const double *inv_freq, size_t tokens, int q_heads, int k_heads, int v_heads,
                                 int head_dim, int rotary_dim, int interleaved, float eps, int dtype, void *stream)
{
    NormCall c = {};
    c.bufs = bufs;
    c.world = world;
    c.out[0] = q_out, c.out[1] = k_out, c.out[2] = v_out;
    c.weight[0] = q_weight, c.weight[1] = k_weight;
    c.positions = positions;
    c.inv_freq = inv_freq;
    c.tokens = tokens;
    c.heads[0] = q_heads, c.heads[1] = k_heads, c.heads[2] = v_heads;
    c.dim = head_dim, c.rotary = rotary_dim, c.interleaved = interleaved;
    c.eps = eps;
    if (const int rc = check_norm(c, dtype)) return rc;
    if (tokens == 0) return TCCL_OK;
    c.tokens_per_wg = norm_tokens_per_wg(c);
    c.workgroups = norm_workgroups(c);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return hip_code(dtype == TCCL_BF16 ? launch_norm_dim<Bf16Row>(c, s) : launch_norm_dim<F32Row>(c, s));
}

extern "C" size_t tccl_qk_norm_rope_backward_workspace(int head_dim)
{
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return 0;
    return static_cast<size_t>(compute_units()) * kMostGradPerUnit * 2 * head_dim * sizeof(float);
}

extern "C" int tccl_qk_norm_rope_backward(const void *const *bufs, int world, const void *dq, const void *dk,
                                          const void *dv, const void *q_weight, const void *k_weight,
                                          const int64_t *positions, const double *inv_freq, void *dx,
                                          float *dq_weight, float *dk_weight, void *workspace, size_t workspace_bytes,
                                          size_t tokens, int q_heads, int k_heads, int v_heads, int head_dim,
                                          int rotary_dim, int interleaved, float eps, int dtype, void *stream)
{
    NormCall c = {};
    c.backward = true;
    c.bufs = bufs;
    c.world = world;
    c.out[0] = dx;
    c.grad[0] = dq, c.grad[1] = dk, c.grad[2] = dv;
    c.weight[0] = q_weight, c.weight[1] = k_weight;
    c.positions = positions;
    c.inv_freq = inv_freq;
    c.partial = static_cast<float *>(workspace);
    c.tokens = tokens;
    c.heads[0] = q_heads, c.heads[1] = k_heads, c.heads[2] = v_heads;
    c.dim = head_dim, c.rotary = rotary_dim, c.interleaved = interleaved;
    c.eps = eps;
    if (const int rc = check_norm(c, dtype)) return rc;
    if (dx == nullptr || dq_weight == nullptr || dk_weight == nullptr || workspace == nullptr) return TCCL_EINVAL;
    if (!aligned16(dq_weight) || !aligned16(dk_weight) || !aligned16(workspace)) return TCCL_EALIGN;
    if (workspace_bytes < tccl_qk_norm_rope_backward_workspace(head_dim)) return TCCL_ESCRATCH;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (tokens > 0) {
        c.tokens_per_wg = norm_tokens_per_wg(c);
        c.workgroups = norm_workgroups(c);
        const hipError_t e = dtype == TCCL_BF16 ? launch_norm_dim<Bf16Row>(c, s) : launch_norm_dim<F32Row>(c, s);
        if (e != hipSuccess) return hip_code(e);
    }
    // no tokens: no partial rows, and the weight gradients are zero
    hipLaunchKernelGGL(weight_grad_kernel, dim3(2 * head_dim / 16), dim3(16 * kGradRows), 0, s, c.partial,
                       static_cast<int>(c.workgroups), head_dim, dq_weight, dk_weight);
    return hip_code(hipGetLastError());
}

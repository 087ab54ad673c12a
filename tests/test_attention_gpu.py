"""The attention operators on the GPU against their definitions in 64 bits (oracle.attention_ref).

Tolerances.  u = 2^-24 is half a step of fp32.  A result rounded once to a type of half-step h is off by h |value| plus
what fp32 arithmetic before it was off; each fp32 operation adds at most u times its result, so a value formed by K
operations from terms of magnitude at most M is off by at most K u M.  K is counted per operator below and stands beside
its bound; v_rsq, v_exp, v_log, cos and sin are off by at most a few steps and count as 4."""
import gc
import math

import pytest
import torch

import tccl_amd
from oracle import attention_ref as ref
from helpers import assert_bit_equal, bits

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.fixture(autouse=True)
def _gpu_hygiene():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    tccl_amd.load_library()
    yield
    torch.cuda.synchronize()
    gc.collect()
    torch.cuda.empty_cache()


def within(got, want, tolerance, what=""):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    off = torch.where(same, 0.0, (got - want).abs())
    worst = (off / torch.as_tensor(tolerance, dtype=torch.float64).clamp(min=1e-300)).max().item() if got.numel() else 0.0
    print(f"{what}: {worst:.3f} of the tolerance")
    assert worst <= 1.0, f"{what}: {worst} times the tolerance"       # a NaN on one side only is not <= 1 either


def world_of(parts):
    group = tccl_amd.empty_world(len(parts), tuple(parts[0].shape), parts[0].dtype, DEV)
    for r, p in enumerate(parts):
        group.tensor(r).copy_(p)
    return group


# ---------------------------------------------------------------- sum, norm and rotation

def norm_inputs(world, tokens, heads, dim, rotary, dtype, far=200_000, seed=0):
    rng = torch.Generator().manual_seed(seed)
    parts = [torch.randn(tokens, sum(heads) * dim, generator=rng).to(dtype) for _ in range(world)]
    w = [(1 + 0.3 * torch.randn(dim, generator=rng)).to(dtype) for _ in range(2)]
    positions = torch.randint(0, far, (tokens,), generator=rng)
    inv_freq = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / max(rotary, 1))
    grads = [torch.randn(tokens, n, dim, generator=rng).to(dtype) for n in heads]
    return parts, w, positions, inv_freq, grads


def row_max(x):
    return x.abs().amax(-1, keepdim=True)


def check_forward(got, parts, w, positions, inv_freq, heads, eps, interleaved):
    dim, dtype, world = w[0].numel(), parts[0].dtype, len(parts)
    x, absolute = sum(p.double() for p in parts), sum(p.double().abs() for p in parts)
    want = ref.qk_norm_rope(x, w[0].double(), w[1].double(), positions, inv_freq, heads[0], heads[1], eps, interleaved)
    split = [t.double() for t in x.view(x.shape[0], -1, dim).tensor_split((heads[0], heads[0] + heads[1]), 1)]
    magnitude = [t for t in absolute.view(x.shape[0], -1, dim).tensor_split((heads[0], heads[0] + heads[1]), 1)]
    for i, name in enumerate("qkv"):
        if want[i].numel() == 0:
            assert got[i].shape == want[i].shape
            continue
        m = row_max(magnitude[i])
        if i < 2:
            # 1 / sqrt(mean x^2): an error d of each x of a row moves the mean's root by at most max d, relative to the root
            r = 1 / torch.sqrt(split[i].square().mean(-1, keepdim=True) + eps)
            worst = row_max(magnitude[i] * r)
            m = m * r * row_max(w[i].double()[None, None]) * (1 + worst) * 2     # two terms of a rotated pair
        # world adds; 8 + 5 adds and 4 in the mean, 4 in rsqrt, 2 products, 3 in the rotation with cos and sin off by 4
        bound = half_step(dtype) * want[i].abs() * (1 + 2.0 ** -7) + (world + 32) * U * m
        within(got[i], want[i], bound, f"{name} w{world} {tuple(want[i].shape)} {dtype}")


NORM_CASES = [
    # world, tokens, heads, dim, rotary, interleaved, dtype
    (1, 1, (1, 0, 0), 64, 64, False, BF16),
    (2, 1, (1, 1, 1), 256, 256, True, BF16),
    (3, 5, (3, 1, 0), 128, 128, False, F32),
    (8, 33, (32, 8, 8), 128, 128, False, BF16),
    (4, 17, (5, 5, 5), 64, 32, True, F32),
    (5, 7, (0, 3, 2), 128, 16, False, BF16),
    (6, 9, (7, 1, 1), 256, 48, False, F32),
    (7, 3, (2, 2, 0), 64, 0, False, BF16),
    (8, 6, (2, 1, 1), 256, 128, True, F32),
    (1, 1027, (4, 2, 2), 64, 64, True, BF16),
    (1, 130, (40, 8, 8), 128, 64, False, F32),
    (2, 2048, (1, 1, 1), 64, 16, True, F32),
]


@pytest.mark.parametrize("case", NORM_CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_qk_norm_rope(case):
    world, tokens, heads, dim, rotary, interleaved, dtype = case
    parts, w, positions, inv_freq, _ = norm_inputs(world, tokens, heads, dim, rotary, dtype)
    group = world_of(parts)
    dw = [t.to(DEV) for t in w]
    rank = world - 1
    got = tccl_amd.qk_norm_rope(group.tensor(rank), *dw, positions.to(DEV), inv_freq.to(DEV), heads[0], heads[1], interleaved=interleaved)
    assert all(g.dtype == dtype for g in got)
    check_forward(got, parts, w, positions, inv_freq, heads, 1e-6, interleaved)
    # value heads are the all-reduce's own columns, bit for bit
    if heads[2] and (tokens * sum(heads) * dim) % 4 == 0:
        summed = tccl_amd.one_shot_all_reduce(group.tensor(0)).view(tokens, -1, dim)
        assert_bit_equal(got[2], summed[:, heads[0] + heads[1]:].contiguous(), "v against the all-reduce")


@pytest.mark.parametrize("case", NORM_CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_qk_norm_rope_backward(case):
    world, tokens, heads, dim, rotary, interleaved, dtype = case
    parts, w, positions, inv_freq, grads = norm_inputs(world, tokens, heads, dim, rotary, dtype, seed=1)
    group = world_of(parts)
    got = tccl_amd.qk_norm_rope_backward(*(g.to(DEV) for g in grads), group.tensor(0), w[0].to(DEV), w[1].to(DEV), positions.to(DEV),
                                         inv_freq.to(DEV), interleaved=interleaved)
    again = tccl_amd.qk_norm_rope_backward(*(g.to(DEV) for g in grads), group.tensor(world - 1), w[0].to(DEV), w[1].to(DEV),
                                           positions.to(DEV), inv_freq.to(DEV), interleaved=interleaved)
    for a, b in zip(got, again):
        assert_bit_equal(a, b, "the same call twice")
    want = ref.qk_norm_rope_grad(parts, grads, *w, positions, inv_freq, 1e-6, interleaved)
    x = sum(p.double() for p in parts).view(tokens, -1, dim)
    absolute = sum(p.double().abs() for p in parts).view(tokens, -1, dim)
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    n = absolute * r
    weight = torch.cat([torch.ones(tokens, heads[i], dim, dtype=torch.float64) * (w[i].double() if i < 2 else 1) for i in range(3)], 1)
    dy = torch.cat([g.double() for g in grads], 1)
    g = 2 * row_max(dy)                                              # a rotated pair
    # dx = r (u - n mean(u n)): both terms at most r max|u| (1 + max n^2); the errors of x move n by (1 + max n) of them
    m = r * g * row_max(weight) * (1 + row_max(n) ** 2) * (1 + row_max(n))
    m[:, heads[0] + heads[1]:] = row_max(dy)[:, heads[0] + heads[1]:] * 0
    # world adds, 32 as in the forward pass, 13 + 4 of the second mean and 4 of the last line
    within(got[0].view(tokens, -1, dim), want[0].view(tokens, -1, dim),
           half_step(dtype) * want[0].view(tokens, -1, dim).abs() * (1 + 2.0 ** -7) + (world + 56) * U * m, f"dx w{world} {dtype}")
    for i, name in enumerate(("dq_weight", "dk_weight")):
        part = slice(0, heads[0]) if i == 0 else slice(heads[0], heads[0] + heads[1])
        terms = (g[:, part] * n[:, part] * (1 + row_max(n[:, part]))).sum((0, 1))
        # a lane adds at most one term per head of the tokens that its workgroup takes (these tests have at most 4,096, one round
        # of workgroups), then 6 + 4 parts of its workgroup, then of at most 1,280 workgroups every 64th, 16 and 4 of those
        chain = sum(heads) * -(-tokens // 4096) + 10 + 20 + 20
        assert got[1 + i].dtype == F32
        within(got[1 + i], want[1 + i], (chain + world + 64) * U * terms, name)


def check_backward(got, parts, w, positions, inv_freq, grads, heads, eps, interleaved, per_lane):
    """`per_lane`: how many terms of a weight's gradient a lane adds up at most.  The counts are those of
    test_qk_norm_rope_backward; eps in the root makes every factor smaller, except that 1 / sqrt(mean x^2 + eps) then moves by
    less than an error of x, which the bounds do not use."""
    world, tokens, dim, dtype = len(parts), parts[0].shape[0], w[0].numel(), parts[0].dtype
    want = ref.qk_norm_rope_grad(parts, grads, *w, positions, inv_freq, eps, interleaved)
    x = sum(p.double() for p in parts).view(tokens, -1, dim)
    absolute = sum(p.double().abs() for p in parts).view(tokens, -1, dim)
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    n = absolute * r
    weight = torch.cat([torch.ones(tokens, heads[i], dim, dtype=torch.float64) * (w[i].double() if i < 2 else 1) for i in range(3)], 1)
    g = 2 * row_max(torch.cat([t.double() for t in grads], 1))       # a rotated pair
    m = r * g * row_max(weight) * (1 + row_max(n) ** 2) * (1 + row_max(n))
    m[:, heads[0] + heads[1]:] = 0
    dx, want_dx = got[0].view(tokens, -1, dim), want[0].view(tokens, -1, dim)
    within(dx, want_dx, half_step(dtype) * want_dx.abs() * (1 + 2.0 ** -7) + (world + 56) * U * m, f"dx w{world} eps {eps}")
    for i, name in enumerate(("dq_weight", "dk_weight")):
        part = slice(0, heads[0]) if i == 0 else slice(heads[0], heads[0] + heads[1])
        terms = (g[:, part] * n[:, part] * (1 + row_max(n[:, part]))).sum((0, 1))
        within(got[1 + i], want[1 + i], (per_lane + 50 + world + 64) * U * terms, f"{name} eps {eps}")


EPS_CASES = [
    # world, tokens, heads, dim, rotary, interleaved, dtype: what of a wave has no work
    (1, 5, (3, 1, 1), 64, 64, False, F32),       # the last workgroup has one token of four; heads of every kind in one wave
    (2, 6, (3, 0, 0), 64, 32, True, BF16),        # query heads only, five places of eight without a head
    (1, 7, (12, 0, 0), 64, 64, False, F32),       # two waves of heads per token, the second half empty, one token of two missing
    (3, 9, (16, 3, 0), 128, 128, False, BF16),    # the keys' wave has one place without a head
    (1, 3, (0, 5, 0), 256, 48, False, F32),
    (2, 3, (2, 2, 3), 128, 0, False, F32),        # queries and keys fill a wave, the values' wave is cut
    (1, 9, (8, 4, 1), 64, 16, True, BF16),        # keys, a value and empty places in one wave
]


@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-2, 100.0])
@pytest.mark.parametrize("case", EPS_CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_qk_norm_rope_any_eps_with_heads_and_tokens_missing(case, eps):
    """Rows that are not zero have a norm and gradients for eps = 0 too; lanes without a head or a token add nothing to them."""
    world, tokens, heads, dim, rotary, interleaved, dtype = case
    parts, w, positions, inv_freq, grads = norm_inputs(world, tokens, heads, dim, rotary, dtype, seed=2)
    group = world_of(parts)
    dev = [t.to(DEV) for t in (*w, positions, inv_freq)]
    got = tccl_amd.qk_norm_rope(group.tensor(0), *dev, heads[0], heads[1], eps=eps, interleaved=interleaved)
    check_forward(got, parts, w, positions, inv_freq, heads, eps, interleaved)
    got = tccl_amd.qk_norm_rope_backward(*(g.to(DEV) for g in grads), group.tensor(0), *dev, eps=eps, interleaved=interleaved)
    check_backward(got, parts, w, positions, inv_freq, grads, heads, eps, interleaved, sum(heads))


ROUND_CASES = [
    # world, tokens, heads, dim, rotary, interleaved, dtype, tokens per workgroup (a wave's share of heads: 512 elements)
    (1, 4099, (16, 8, 8), 64, 64, False, BF16, 1),
    (1, 2600, (10, 5, 0), 128, 32, True, F32, 1),
    (8, 2600, (12, 6, 7), 64, 64, True, F32, 1),
    (2, 4003, (4, 2, 1), 128, 128, False, BF16, 2),
    (2, 13_003, (3, 1, 1), 64, 16, False, F32, 4),
]


@pytest.mark.parametrize("case", ROUND_CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_qk_norm_rope_backward_over_several_rounds_of_tokens(case):
    """More tokens than the workgroups that run at once (five per compute unit at most) take: each walks on with the grid's stride,
    writes other angles into the same LDS and keeps its sums."""
    world, tokens, heads, dim, rotary, interleaved, dtype, at_once = case
    workgroups = -(-tokens // at_once)
    least = torch.cuda.get_device_properties(0).multi_processor_count * 3          # of the eight-source fp32 kernel
    most = least // 3 * (3 if world > 6 else 4 if dtype == F32 else 5)
    assert workgroups > most
    parts, w, positions, inv_freq, grads = norm_inputs(world, tokens, heads, dim, rotary, dtype, seed=tokens)
    group = world_of(parts)
    dev = [t.to(DEV) for t in (*w, positions, inv_freq)]
    got = tccl_amd.qk_norm_rope_backward(*(g.to(DEV) for g in grads), group.tensor(0), *dev, interleaved=interleaved)
    rounds = -(-workgroups // least)
    check_backward(got, parts, w, positions, inv_freq, grads, heads, 1e-6, interleaved, sum(heads) * at_once * rounds)
    again = tccl_amd.qk_norm_rope_backward(*(g.to(DEV) for g in grads), group.tensor(0), *dev, interleaved=interleaved)
    for a, b in zip(got, again):
        assert_bit_equal(a, b, "the same call twice")


def test_qk_norm_rope_backward_against_differences():
    """<dx, d> and <dw, d> in float32 against differences of the 64-bit forward pass."""
    heads, dim, tokens = (3, 2, 1), 128, 6
    parts, w, positions, inv_freq, grads = norm_inputs(2, tokens, heads, dim, 128, F32, far=5000, seed=4)
    group = world_of(parts)
    dx, dqw, dkw = tccl_amd.qk_norm_rope_backward(*(g.to(DEV) for g in grads), group.tensor(0), w[0].to(DEV), w[1].to(DEV),
                                                  positions.to(DEV), inv_freq.to(DEV))

    def value(x, qw, kw):
        y = ref.qk_norm_rope(x, qw, kw, positions, inv_freq, heads[0], heads[1], 1e-6, False)
        return sum((a * g.double()).sum() for a, g in zip(y, grads)).item()

    at = [sum(p.double() for p in parts), w[0].double(), w[1].double()]
    h = 1e-5
    for i, got in enumerate((dx, dqw, dkw)):
        d = torch.randn(at[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + h * d, at[i] - h * d
        numeric = (value(*up) - value(*down)) / (2 * h)
        terms = (got.cpu().double().view_as(d) * d)
        # fp32 gradients are off by under 100 u of their terms' magnitude, the difference by h^2 of a third derivative of the same order
        assert abs(numeric - terms.sum().item()) <= (100 * U + 1e-8) * 30 * terms.abs().sum().item()


def test_qk_norm_rope_far_positions_and_negative_ones():
    heads, dim = (2, 1, 0), 128
    parts, w, _, inv_freq, _ = norm_inputs(1, 6, heads, dim, 128, F32, seed=7)
    positions = torch.tensor([0, 1, -5, 1 << 24, 10_000_019, (1 << 31) + 3])
    got = tccl_amd.qk_norm_rope(world_of(parts).tensor(0), w[0].to(DEV), w[1].to(DEV), positions.to(DEV), inv_freq.to(DEV), 2, 1)
    # an fp64 angle of 2^31 is off by 2^-22 of a step of 1, which is far above what fp32 rounds: compare up to 2^24 closely
    near = slice(0, 5)
    check_forward([t[near] for t in got], [parts[0][near]], w, positions[near], inv_freq, heads, 1e-6, False)
    want = ref.qk_norm_rope(parts[0].double(), w[0].double(), w[1].double(), positions, inv_freq, 2, 1, 1e-6, False)
    within(got[0][5:], want[0][5:], 2.0 ** -18 * row_max(want[0][5:]) * 2, "position 2^31")


def test_qk_norm_rope_special_values():
    """A row of zeros stays zero, a NaN or an infinity stays in its own head."""
    heads, dim = (3, 1, 1), 64
    parts, w, positions, inv_freq, _ = norm_inputs(1, 4, heads, dim, 64, F32, seed=9)
    x = parts[0].view(4, 5, dim)
    x[0, 0] = 0
    x[1, 1, 5] = math.nan
    x[2, 3, 7] = math.inf
    x[3, 2] *= 1e-30
    x[3, 4, 0] = math.inf
    got = tccl_amd.qk_norm_rope(world_of(parts).tensor(0), w[0].to(DEV), w[1].to(DEV), positions.to(DEV), inv_freq.to(DEV), 3, 1)
    q, k, v = (t.cpu() for t in got)
    assert torch.equal(q[0, 0], torch.zeros(dim))
    assert torch.isnan(q[1, 1]).all() and torch.isfinite(q[1, 0]).all() and torch.isfinite(q[1, 2]).all()
    assert not torch.isfinite(k[2, 0]).all() and torch.isfinite(q[2]).all()
    assert torch.isfinite(q[3, 2]).all() and v[3, 0, 0] == math.inf and torch.isfinite(v[3, 0, 1:]).all()


@pytest.mark.parametrize("power", [-60, 0, 58])
def test_qk_norm_rope_of_small_and_large_rows(power):
    """Every size of row whose sum of squares fp32 holds is normed as well as any other, forward and backward, for eps = 0."""
    heads, dim = (3, 1, 1), 64
    parts, w, positions, inv_freq, grads = norm_inputs(1, 5, heads, dim, dim, F32, seed=19)
    parts = [p * 2.0 ** power for p in parts]
    group = world_of(parts)
    dev = [t.to(DEV) for t in (*w, positions, inv_freq)]
    check_forward(tccl_amd.qk_norm_rope(group.tensor(0), *dev, 3, 1, eps=0.0), parts, w, positions, inv_freq, heads, 0.0, False)
    got = tccl_amd.qk_norm_rope_backward(*(g.to(DEV) for g in grads), group.tensor(0), *dev, eps=0.0)
    check_backward(got, parts, w, positions, inv_freq, grads, heads, 0.0, False, sum(heads))


def test_qk_norm_rope_of_rows_beyond_fp32():
    parts, w, positions, inv_freq, grads = norm_inputs(1, 3, (2, 1, 0), 64, 64, F32, seed=20)
    x = parts[0].view(3, 3, 64)
    x[1, 1] *= 2.0 ** 70
    group = world_of(parts)
    dev = [t.to(DEV) for t in (*w, positions, inv_freq)]
    q, _, _ = tccl_amd.qk_norm_rope(group.tensor(0), *dev, 2, 1)
    assert not q[1, 1].any() and q[1, 0].any() and torch.isfinite(q).all()
    got = tccl_amd.qk_norm_rope_backward(*(g.to(DEV) for g in grads), group.tensor(0), *dev)
    assert not got[0].view(3, 3, 64)[1, 1].any() and all(torch.isfinite(t).all() for t in got)


def test_norm_without_tokens_and_with_a_prefix_view():
    parts, w, positions, inv_freq, _ = norm_inputs(2, 8, (2, 1, 1), 64, 64, BF16)
    group = world_of(parts)
    dw = [t.to(DEV) for t in w]
    q, k, v = tccl_amd.qk_norm_rope(group.tensor(0)[:0], *dw, positions[:0].to(DEV), inv_freq.to(DEV), 2, 1)
    assert q.shape == (0, 2, 64) and v.shape == (0, 1, 64)
    dx, dqw, dkw = tccl_amd.qk_norm_rope_backward(q, k, v, group.tensor(0)[:0], *dw, positions[:0].to(DEV), inv_freq.to(DEV))
    assert dx.shape == (0, 256) and not dqw.any() and not dkw.any()
    got = tccl_amd.qk_norm_rope(group.tensor(1)[:5], *dw, positions.to(DEV)[:5], inv_freq.to(DEV), 2, 1)
    check_forward(got, [p[:5] for p in parts], w, positions[:5], inv_freq, (2, 1, 1), 1e-6, False)


def test_norm_of_buffers_behind_four_gib():
    """Offsets that pass 32 bits, in elements and in bytes: only the last tokens are other than zero, and carry gradients."""
    heads, dim, some = (20, 4, 4), 128, 5
    columns = sum(heads) * dim
    tokens = (9 << 30) // (2 * columns) | 1                              # 4.8e9 elements
    last, w, _, inv_freq, grads = norm_inputs(1, some, heads, dim, dim, BF16, seed=17)
    positions = torch.arange(tokens)
    x = torch.zeros(tokens, columns, dtype=BF16, device=DEV)
    x[-some:] = last[0].to(DEV)
    group = tccl_amd.register([x])
    dev = [t.to(DEV) for t in (*w, positions, inv_freq)]
    got = tccl_amd.qk_norm_rope(x, *dev, heads[0], heads[1])
    check_forward([t[-some:] for t in got], last, w, positions[-some:], inv_freq, heads, 1e-6, False)
    assert not any(t[:1000].any() or t[-some - 1000:-some].any() for t in got)
    for t, g in zip(got, grads):
        t.zero_()
        t[-some:] = g.to(DEV)
    dx, *dw = tccl_amd.qk_norm_rope_backward(*got, x, *dev)
    check_backward([dx[-some:], *dw], last, w, positions[-some:], inv_freq, grads, heads, 1e-6, False, some * sum(heads))
    assert not dx[:1000].any() and not dx[-some - 1000:-some].any()
    tccl_amd.unregister(group)


# ---------------------------------------------------------------- the paged cache

def read_back(cache, slots, dtype=BF16):
    k, v = tccl_amd.cache_read(cache, slots.to(DEV), dtype=dtype)
    return k.cpu(), v.cpu()


def assert_stored(got, x, store, what):
    want = ref.stored(x, store)
    g = got.double()
    same = (g == want) | (torch.isnan(g) & torch.isnan(want))
    assert same.all(), f"{what}: {(~same).sum().item()} of {g.numel()} values differ"


CACHE_CASES = [
    # world, pages per rank, page, heads, dim, store, source
    (1, 4, 16, 1, 64, BF16, BF16),
    (2, 3, 32, 3, 128, E4M3, BF16),
    (8, 2, 64, 2, 256, E4M3, F32),
    (3, 2, 128, 4, 64, E4M3, BF16),
    (4, 1, 256, 1, 128, BF16, F32),
    (5, 5, 16, 2, 256, BF16, BF16),
    (1, 9, 16, 8, 64, E4M3, F32),
    # enough tokens for the larger tiles
    (8, 40, 64, 8, 64, E4M3, BF16),
    (4, 70, 128, 4, 128, BF16, BF16),
    (2, 50, 256, 2, 256, E4M3, F32),
    (1, 700, 16, 6, 64, BF16, F32),
    (3, 200, 32, 2, 128, E4M3, F32),
]


@pytest.mark.parametrize("order", ["runs", "shuffled"])
@pytest.mark.parametrize("case", CACHE_CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_cache_write_and_read(case, order):
    world, pages, page, heads, dim, store, dtype = case
    cache = tccl_amd.PagedCache(world, pages, page, heads, dim, dtype=store, device=DEV)
    rng = torch.Generator().manual_seed(5)
    # every third page is left alone; runs start anywhere in a page, and some entries of the list are padding
    slots = torch.arange(cache.slots)
    slots = slots[(slots // page) % 3 != 2]
    slots = slots[5:-3]
    if order == "shuffled":
        slots = slots[torch.randperm(len(slots), generator=rng)]
    slots[7::13] = -1
    slots[3] = cache.slots                                     # one behind the pool
    x = [torch.randn(len(slots), heads, dim, generator=rng).to(dtype) for _ in range(2)]
    tccl_amd.cache_write(cache, x[0].to(DEV), x[1].to(DEV), slots.to(DEV))
    k, v = read_back(cache, torch.arange(cache.slots), dtype)
    written = (slots >= 0) & (slots < cache.slots)
    at = slots[written]
    assert_stored(k[at], x[0][written], store, "k")
    assert_stored(v[at], x[1][written], store, "v")
    rest = torch.ones(cache.slots, dtype=torch.bool)
    rest[at] = False
    assert not k[rest].any() and not v[rest].any(), "slots that were not written"
    # read in the list's own order: padding reads as zeros, repeats are allowed
    again = torch.cat((slots, slots[:20]))
    k2, v2 = read_back(cache, again, F32)
    ok = (again >= 0) & (again < cache.slots)
    assert torch.equal(k2[ok], k[again[ok]].float()) and torch.equal(v2[ok], v[again[ok]].float())
    assert not k2[~ok].any() and not v2[~ok].any()


@pytest.mark.parametrize("store", [BF16, E4M3])
def test_cache_special_rows(store):
    """Zero rows, a tiny row, the largest finite values, infinities and NaN: each touches its own row only."""
    dim = 64
    cache = tccl_amd.PagedCache(2, 2, 16, 1, dim, dtype=store, device=DEV)
    x = torch.randn(9, 1, dim, generator=torch.Generator().manual_seed(2))
    x[0] = 0
    x[1] *= 1e-36
    x[2] *= 1e30
    x[3, 0, 5] = math.nan
    x[4, 0, 6] = math.inf
    x[5] = math.inf
    x[6, 0, 0], x[6, 0, 1] = 448.0, -448.0
    x[7, 0, 0] = 449.0
    x[8, 0, 3] = -0.0
    slots = torch.arange(9) + 3
    tccl_amd.cache_write(cache, x.to(DEV), x.to(DEV), slots.to(DEV))
    k, v = read_back(cache, slots, F32)
    if store == BF16:
        want = x.to(BF16).float()
        assert torch.equal(torch.isnan(k), torch.isnan(want)) and torch.equal(torch.nan_to_num(k), torch.nan_to_num(want))
    else:
        assert_stored(k, x, store, "k")
    assert torch.equal(bits(k), bits(v))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_cache_keeps_the_largest_finite_rows_finite_in_8_bits(dtype):
    """Rows up to the type's largest number: the largest exponent's codes stop where a larger one would stand for 2^128."""
    dim, top = 64, torch.finfo(dtype).max
    largest = torch.tensor([1.75 * 2.0 ** 127, 1.78125 * 2.0 ** 127, 1.921875 * 2.0 ** 127, 1.9375 * 2.0 ** 127, -1.9375 * 2.0 ** 127,
                            1.953125 * 2.0 ** 127, top, -top], dtype=torch.float64)
    x = torch.randn(3 * len(largest), 1, dim, generator=torch.Generator().manual_seed(6)) * 1e37
    x[:, 0, 5] = largest.repeat(3).float()
    x[8:16, 0, 9], x[8:16, 0, 10] = math.nan, -math.inf       # beside what is not finite
    x[16:, 0, 20:40] = largest[:, None].float() * torch.linspace(0.9, 1, 20)
    x = x.to(dtype)
    assert torch.isfinite(x[:8]).all() and torch.isfinite(x[16:]).all()
    cache = tccl_amd.PagedCache(2, 2, 16, 1, dim, dtype=E4M3, device=DEV)
    slots = torch.arange(len(x)) + 3
    tccl_amd.cache_write(cache, x.to(DEV), x.flip(0).to(DEV), slots.to(DEV))
    for as_dtype in (BF16, F32):
        k, v = read_back(cache, slots, as_dtype)
        assert_stored(k, x, E4M3, "k")
        assert_stored(v, x.flip(0), E4M3, "v")
        assert torch.isfinite(k[:8]).all() and torch.isfinite(k[16:]).all()
    # a sequence of one token returns the token's values as they are kept
    table, n = torch.tensor([[0]], dtype=torch.int32, device=DEV), torch.tensor([1], dtype=torch.int32, device=DEV)
    for t in (0, 3, 6, 7):
        tccl_amd.cache_write(cache, torch.zeros_like(x[:1]).to(DEV), x[t: t + 1].to(DEV), torch.tensor([0], device=DEV))
        out = tccl_amd.decode_attention(torch.ones(1, 1, dim, dtype=BF16, device=DEV), cache, table, n)
        assert torch.equal(out[0].cpu().double(), ref.stored(x[t], E4M3)), t


def test_cache_takes_strided_sources():
    """k and v as views of one projection's rows, and a head-major tensor."""
    heads, dim, tokens = 3, 128, 50
    cache = tccl_amd.PagedCache(2, 4, 16, heads, dim, dtype=E4M3, device=DEV)
    qkv = torch.randn(tokens, 4 * heads, dim, generator=torch.Generator().manual_seed(8)).to(BF16)
    on = qkv.to(DEV)
    slots = torch.arange(tokens) + 9
    tccl_amd.cache_write(cache, on[:, heads:2 * heads], on[:, 2 * heads:3 * heads], slots.to(DEV))
    k, v = read_back(cache, slots)
    assert_stored(k, qkv[:, heads:2 * heads], E4M3, "k")
    assert_stored(v, qkv[:, 2 * heads:3 * heads], E4M3, "v")
    swapped = on[:, :heads].transpose(0, 1).contiguous().transpose(0, 1)
    one = on[:, :1].expand(tokens, heads, dim)                                # one head for all: a stride of 0
    tccl_amd.cache_write(cache, swapped, one, slots.to(DEV))
    k, v = read_back(cache, slots)
    assert_stored(k, qkv[:, :heads], E4M3, "k")
    assert_stored(v, qkv[:, :1].expand(tokens, heads, dim), E4M3, "v")


@pytest.mark.parametrize("store", [BF16, E4M3])
def test_cache_behind_four_gib(store):
    """Offsets into one rank's buffer that pass 32 bits; attention over the same pages."""
    dim, heads, page = 128, 8, 256
    block = page * dim * 2 * (2 if store == BF16 else 1) + (0 if store == BF16 else 2 * page)
    pages = (5 << 30) // (block * heads)
    cache = tccl_amd.PagedCache(1, pages, page, heads, dim, dtype=store, device=DEV)
    rng = torch.Generator().manual_seed(3)
    x = [torch.randn(300, heads, dim, generator=rng).to(BF16) for _ in range(2)]
    table = torch.tensor([[pages - 1, pages - 7]], dtype=torch.int32)
    t = torch.arange(300)
    slots = table[0].long()[t // page] * page + t % page
    tccl_amd.cache_write(cache, x[0].to(DEV), x[1].to(DEV), slots.to(DEV))
    k, v = read_back(cache, slots)
    assert_stored(k, x[0], store, "k")
    assert_stored(v, x[1], store, "v")
    q = torch.randn(1, heads * 2, dim, generator=rng).to(BF16)
    out, lse = tccl_amd.decode_attention(q.to(DEV), cache, table.to(DEV), torch.tensor([300], dtype=torch.int32, device=DEV), return_lse=True)
    check_attention(out, lse, q, [k.double()], [v.double()])


@pytest.mark.parametrize("store", [BF16, E4M3])
def test_cache_far_slots_and_given_outputs(store):
    """Slots at both ends of int64 are padding; outputs that the caller gives are filled whole and nothing beside them."""
    heads, dim = 2, 64
    cache = tccl_amd.PagedCache(2, 3, 32, heads, dim, dtype=store, device=DEV)
    x = torch.randn(6, heads, dim, generator=torch.Generator().manual_seed(14)).to(BF16)
    slots = torch.tensor([-2 ** 63, 70, 2 ** 63 - 1, 71, cache.slots, 2 ** 40])
    tccl_amd.cache_write(cache, x.to(DEV), x.to(DEV), slots.to(DEV))
    for dtype in (BF16, F32):
        wide = torch.full((3, 8, heads, dim), 9.0, dtype=dtype, device=DEV)
        got = tccl_amd.cache_read(cache, slots.to(DEV), dtype=dtype, out=(wide[0, 1:7], wide[2, :6]))
        assert got[0].data_ptr() == wide[0, 1].data_ptr() and got[1].data_ptr() == wide[2].data_ptr()
        for t in got:
            assert_stored(t.cpu()[1::2][:2], x[1::2][:2], store, "written")
            assert not t[::2].any() and not t[5].any()
        assert (wide[1] == 9).all() and (wide[0, 0] == 9).all() and (wide[0, 7] == 9).all() and (wide[2, 6:] == 9).all()
    everything = tccl_amd.cache_read(cache, torch.arange(cache.slots, device=DEV))
    assert sorted(torch.nonzero(everything[0].any(-1).any(-1))[:, 0].tolist()) == [70, 71]


def test_cache_without_tokens():
    cache = tccl_amd.PagedCache(1, 1, 16, 2, 64, device=DEV)
    none = torch.empty(0, 2, 64, device=DEV)
    tccl_amd.cache_write(cache, none, none, torch.empty(0, dtype=torch.int64, device=DEV))
    k, v = tccl_amd.cache_read(cache, torch.empty(0, dtype=torch.int64, device=DEV))
    assert k.shape == v.shape == (0, 2, 64)


# ---------------------------------------------------------------- attention

def check_attention(out, lse, q, keys, values, scale=None, what=""):
    """out is one bf16 rounding of sum p v / sum p.  A score of D products is off by (D + 4) u sum |q k| scale; exp2 of it by twice
    that, 4 u and u |score| of the base change; P as two bf16 terms by 2^-18; the sums over n tokens by (n / 4 + 64) u.  A term that
    is below the smallest normal number, 2^-126, may count as zero: P has two terms per token and sum p is at least 1 (the
    maximum's own), so all of them together move the output by at most 2 n 2^-126."""
    want, want_lse = ref.attention(q, keys, values, scale)
    dim = q.shape[-1]
    scale = 1 / math.sqrt(dim) if scale is None else scale
    bound, bound_lse = torch.zeros_like(want), torch.zeros_like(want_lse)
    for b in range(q.shape[0]):
        n = keys[b].shape[0]
        if n == 0:
            continue
        group = q.shape[1] // keys[b].shape[1]
        for h in range(q.shape[1]):
            kk, vv = keys[b][:, h // group].double(), values[b][:, h // group].double()
            s = kk @ q[b, h].double() * scale
            ds = (dim + 4) * U * (kk.abs() @ q[b, h].double().abs() * abs(scale)).max() + 4 * U * s.abs().max()
            rel = 2 * ds + 2.0 ** -17 + (n / 4 + 80) * U
            bound[b, h] = half_step(BF16) * want[b, h].abs() * (1 + 2.0 ** -7) + rel * (torch.softmax(s, 0) @ vv.abs()) + 2 * n * 2.0 ** -126
            bound_lse[b, h] = 2 * ds + (n / 4 + 80) * U + 4 * U * want_lse[b, h].abs()
    within(out, want, bound, f"out {what}")
    if lse is not None:
        within(lse, want_lse, bound_lse, f"lse {what}")


def filled(world, lengths, q_heads, kv_heads, dim, page, store, seed=0, spare=3, spread=1.0):
    """A cache with sequences on pages in random order over all ranks, garbage on every page that is not written."""
    rng = torch.Generator().manual_seed(seed)
    width = max(1, max(-(-n // page) for n in lengths)) + 1                # a table wider than any sequence needs
    used = [-(-n // page) for n in lengths]
    each = -(-(sum(used) + spare) // world)
    cache = tccl_amd.PagedCache(world, each, page, kv_heads, dim, dtype=store, device=DEV)
    for t in cache.group.tensors:
        t.fill_(0xFF)                                                         # NaN as bf16 and as e4m3, the largest scale byte
    ids = torch.randperm(cache.pages, generator=rng)
    table = torch.full((len(lengths), width), -7, dtype=torch.int32)        # entries behind a sequence are no pages
    table[:, -1] = 2 ** 30
    slots, at = [], 0
    for b, n in enumerate(lengths):
        table[b, : used[b]] = ids[at: at + used[b]].int()
        at += used[b]
        t = torch.arange(n)
        slots.append(table[b].long()[t // page] * page + t % page)
    total = sum(lengths)
    k, v = (torch.randn(total, kv_heads, dim, generator=rng).to(BF16) * spread for _ in range(2))
    q = torch.randn(len(lengths), q_heads, dim, generator=rng).to(BF16)
    if total:
        tccl_amd.cache_write(cache, k.to(DEV), v.to(DEV), torch.cat(slots).to(DEV))
    keys = [ref.stored(x, store) for x in k.split(lengths)]
    values = [ref.stored(x, store) for x in v.split(lengths)]
    return cache, table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), q, keys, values, slots


ATTENTION_CASES = [
    # world, lengths, q_heads, kv_heads, dim, page, store
    (1, [1], 1, 1, 64, 16, BF16),
    (1, [1], 1, 1, 128, 16, E4M3),
    (2, [0, 1, 2, 7, 8, 9, 15, 16, 17], 4, 4, 128, 16, BF16),
    (3, [31, 32, 33, 0, 63, 64, 65, 127, 129], 8, 2, 64, 16, E4M3),
    (8, [255, 256, 257, 511, 513], 6, 2, 128, 32, BF16),
    (8, [255, 256, 257, 511, 513], 6, 2, 128, 32, E4M3),
    (4, [1000, 3, 0, 5001], 16, 1, 128, 64, BF16),
    (4, [1000, 3, 0, 5001], 17, 1, 64, 64, E4M3),
    (5, [700, 1], 32, 1, 256, 128, BF16),
    (5, [700, 1], 24, 2, 256, 256, E4M3),
    (1, [20011], 4, 2, 64, 16, BF16),
    (7, [20011], 7, 1, 128, 16, E4M3),
    (6, [40, 41] * 40, 3, 3, 64, 16, BF16),
    (2, [0, 0, 900, 0, 130, 2, 0], 70, 2, 64, 16, BF16),
    (2, [0, 5, 600, 0, 1300, 2, 0] * 3, 35, 1, 128, 32, E4M3),
    (1, [530, 0] + [3] * 300, 2, 2, 64, 16, E4M3),
    (3, [5, 0, 17, 1] * 1100, 1, 1, 64, 16, BF16),
    (1, [600] + [0, 3] * 2100, 2, 1, 64, 16, BF16),
    (2, [20011] + [0, 1] * 2050, 2, 1, 64, 16, E4M3),
    (2, [600, 3, 0] * 700, 1, 1, 64, 16, BF16),
]


@pytest.mark.parametrize("case", ATTENTION_CASES, ids=lambda c: f"w{c[0]}-n{len(c[1])}x{max(c[1])}-q{c[2]}-k{c[3]}-d{c[4]}-p{c[5]}-{str(c[6])[6:]}")
def test_decode_attention(case):
    world, lengths, q_heads, kv_heads, dim, page, store = case
    cache, table, n, q, keys, values, _ = filled(*case)
    out, lse = tccl_amd.decode_attention(q.to(DEV), cache, table, n, return_lse=True)
    check_attention(out, lse, q, keys, values)
    again, lse_again = tccl_amd.decode_attention(q.to(DEV), cache, table, n, return_lse=True)
    assert_bit_equal(out, again, "twice")
    assert_bit_equal(lse, lse_again, "lse twice")
    # another bound of the lengths gives another split: still within the tolerance
    out, lse = tccl_amd.decode_attention(q.to(DEV), cache, table, n, max_length=max(lengths), return_lse=True)
    check_attention(out, lse, q, keys, values, what="max_length")


WIDE_CASES = [
    # more than 64 query heads on one key head: several workgroups per sequence and key head
    (2, [300, 0, 40], 65, 1, 64, 16, BF16),
    (1, [130, 17], 200, 2, 128, 32, E4M3),
    (3, [90, 1], 100, 1, 256, 64, E4M3),
    (1, [5003, 0, 700], 128, 1, 128, 64, E4M3),
    (4, [3001, 1, 900], 100, 1, 256, 16, BF16),
    (2, [9000, 20], 260, 2, 64, 32, BF16),
    # either side of where a fourth wave begins to help: two and three blocks of 16
    (2, [1500, 33], 32, 1, 128, 16, BF16),
    (2, [1500, 33], 33, 1, 128, 16, E4M3),
    (2, [1500, 33], 64, 1, 64, 16, E4M3),
]


@pytest.mark.parametrize("case", WIDE_CASES, ids=lambda c: f"w{c[0]}-n{len(c[1])}x{max(c[1])}-q{c[2]}-k{c[3]}-d{c[4]}-p{c[5]}-{str(c[6])[6:]}")
def test_decode_attention_many_query_heads_on_a_key_head(case):
    cache, table, n, q, keys, values, _ = filled(*case, seed=8)
    out, lse = tccl_amd.decode_attention(q.to(DEV), cache, table, n, return_lse=True)
    check_attention(out, lse, q, keys, values)
    again, lse_again = tccl_amd.decode_attention(q.to(DEV), cache, table, n, return_lse=True)
    assert_bit_equal(out, again, "twice")
    assert_bit_equal(lse, lse_again, "lse twice")


@pytest.mark.parametrize("store", [BF16, E4M3])
def test_decode_attention_more_pages_than_a_workgroup_looks_up_at_once(store):
    """A workgroup looks 512 page addresses up at a time.  Here each one's even share is over 8,192 tokens of 16 per page, so that it
    looks up again, in the middle of a sequence and after it has gone on to the next; peaked scores make every part count."""
    world, kv_heads, group, dim, page = 2, 8, 2, 64, 16
    shares = 2 * torch.cuda.get_device_properties(0).multi_processor_count
    lengths = [83_001, 0, 79_990, 8_193, 80_000, 1, 77_777, 90_111, 85_003, 81_920, 64_005]
    assert sum(lengths) * kv_heads / shares > 1.2 * 512 * page
    rng = torch.Generator(device=DEV).manual_seed(9)
    used = [-(-n // page) for n in lengths]
    cache = tccl_amd.PagedCache(world, -(-sum(used) // world), page, kv_heads, dim, dtype=store, device=DEV)
    ids = torch.randperm(cache.pages, generator=rng, device=DEV)[: sum(used)].split(used)
    table = torch.full((len(lengths), max(used)), -1, dtype=torch.int32, device=DEV)
    keys, values = [], []
    for b, n in enumerate(lengths):
        table[b, : used[b]] = ids[b].int()
        t = torch.arange(n, device=DEV)
        k, v = (torch.randn(n, kv_heads, dim, generator=rng, device=DEV).to(BF16) for _ in range(2))
        if n:
            tccl_amd.cache_write(cache, k, v, ids[b][t // page] * page + t % page)
        keys.append(k)
        values.append(v)
    q = torch.randn(len(lengths), kv_heads * group, dim, generator=rng, device=DEV).to(BF16)
    out, lse = tccl_amd.decode_attention(q, cache, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), scale=0.6, return_lse=True)
    for b in range(len(lengths)):
        for h in range(b % 3, kv_heads, 3):
            heads = slice(h * group, (h + 1) * group)
            kept = [ref.stored(x[b][:, h: h + 1].cpu(), store) for x in (keys, values)]
            check_attention(out[b: b + 1, heads], lse[b: b + 1, heads], q[b: b + 1, heads].cpu(), [kept[0]], [kept[1]], 0.6, f"{b} {h}")


@pytest.mark.parametrize("store", [BF16, E4M3])
def test_decode_attention_peaked_scores_and_scales(store):
    """Scores far apart (a weight underflows to zero), far below zero, and a caller's scale."""
    cache, table, n, q, keys, values, _ = filled(2, [500, 77], 8, 2, 128, 32, store, seed=3, spread=8.0)
    for scale in (None, 1.0, 0.01, -0.3, 0.0):
        out, lse = tccl_amd.decode_attention(q.to(DEV), cache, table, n, scale=scale, return_lse=True)
        check_attention(out, lse, q, keys, values, scale, what=f"scale {scale}")


@pytest.mark.parametrize("store", [BF16, E4M3])
@pytest.mark.parametrize("spread,scale", [(1e-20, None), (1e15, 1e-30), (1e-36, 1.0)])
def test_decode_attention_tiny_and_huge_cached_values(store, spread, scale):
    cache, table, n, q, keys, values, _ = filled(2, [300, 31], 8, 2, 64, 16, store, seed=5, spread=spread)
    out, lse = tccl_amd.decode_attention(q.to(DEV), cache, table, n, scale=scale, return_lse=True)
    check_attention(out, lse, q, keys, values, scale, what=f"values about {spread}")


def test_decode_attention_nan_in_a_query_stays_in_its_head():
    cache, table, n, q, keys, values, _ = filled(2, [700, 90], 12, 3, 64, 16, E4M3, seed=6)
    q[0, 5, 9], q[1, 2, 0] = math.nan, math.inf
    out, lse = (t.cpu() for t in tccl_amd.decode_attention(q.to(DEV), cache, table, n, return_lse=True))
    bad = torch.zeros(2, 12, dtype=torch.bool)
    bad[0, 5] = bad[1, 2] = True
    assert torch.isnan(out[bad]).all() and torch.isnan(lse[0, 5])
    fine = torch.where(bad[..., None], 0.0, q.double()).to(BF16)
    clean, clean_lse = tccl_amd.decode_attention(fine.to(DEV), cache, table, n, return_lse=True)
    assert_bit_equal(out[~bad], clean.cpu()[~bad], "the other heads")
    assert_bit_equal(lse[~bad], clean_lse.cpu()[~bad], "the other heads' lse")


def test_decode_attention_large_negative_scores_only():
    """Every score of a row far below zero: nothing underflows, since the row's own maximum is taken off."""
    cache, table, n, q, keys, values, slots = filled(1, [40], 1, 1, 64, 16, BF16)
    k = torch.full((40, 1, 64), 100.0)
    v = torch.randn(40, 1, 64, generator=torch.Generator().manual_seed(1)).to(BF16).float()
    tccl_amd.cache_write(cache, k.to(DEV), v.to(DEV), slots[0].to(DEV))
    q = torch.full((1, 1, 64), -100.0).to(BF16)
    out, lse = tccl_amd.decode_attention(q.to(DEV), cache, table, n, return_lse=True)
    check_attention(out, lse, q, [k.double()], [v.double()])


def test_decode_attention_strides_and_outputs():
    cache, table, n, q, keys, values, _ = filled(2, [50, 0, 300], 8, 2, 64, 16, BF16)
    wide = torch.zeros(3, 20, 64, dtype=BF16, device=DEV)
    wide[:, 4:12] = q.to(DEV)
    heads_first = q.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
    big_table = torch.full((3, table.shape[1] + 5), -1, dtype=torch.int32, device=DEV)
    big_table[:, : table.shape[1]] = table
    for queries, t in ((wide[:, 4:12], table), (heads_first, big_table[:, : table.shape[1]])):
        out = torch.full((3, 8, 64), 7.0, dtype=BF16, device=DEV)
        lse = torch.full((3, 8), 7.0, device=DEV)
        got = tccl_amd.decode_attention(queries, cache, t, n, out=out, lse=lse)
        assert got[0] is out and got[1] is lse
        check_attention(out, lse, q, keys, values)
    only = tccl_amd.decode_attention(q.to(DEV), cache, table, n)
    assert_bit_equal(only, out, "without lse")
    # a dimension of one may have any stride
    odd = torch.zeros(8 * 64, dtype=BF16, device=DEV).as_strided((1, 8, 64), (3, 64, 1)).copy_(q[2:].to(DEV))
    alone = tccl_amd.decode_attention(odd, cache, table[2:], n[2:])
    check_attention(alone, None, q[2:], keys[2:], values[2:])
    # one query row for every sequence
    one = q[:1].to(DEV).expand(3, 8, 64)
    check_attention(tccl_amd.decode_attention(one, cache, table, n), None, q[:1].expand(3, 8, 64), keys, values)


def test_decode_attention_bounds_of_lengths():
    """max_length and the table's width bound what is read; negative lengths are empty."""
    cache, table, n, q, keys, values, _ = filled(2, [90, 300, 20], 4, 2, 64, 16, E4M3)
    out, lse = tccl_amd.decode_attention(q.to(DEV), cache, table, n, max_length=37, return_lse=True)
    check_attention(out, lse, q, [x[:37] for x in keys], [x[:37] for x in values], what="cut at 37")
    out, lse = tccl_amd.decode_attention(q.to(DEV), cache, table[:, :2].contiguous(), n, return_lse=True)
    check_attention(out, lse, q, [x[:32] for x in keys], [x[:32] for x in values], what="a table of two pages")
    for empty in (dict(max_length=0), {}):
        t = table if empty else table[:, :0]
        out, lse = tccl_amd.decode_attention(q.to(DEV), cache, t, n, return_lse=True, **empty)
        assert not out.any() and (lse == -math.inf).all()
    n[1] = -4
    out, lse = tccl_amd.decode_attention(q.to(DEV), cache, table, n, return_lse=True)
    keys[1], values[1] = keys[1][:0], values[1][:0]
    check_attention(out, lse, q, keys, values, what="a negative length")
    none = tccl_amd.decode_attention(q[:0].to(DEV), cache, table[:0], n[:0])
    assert none.shape == (0, 4, 64)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("store", [BF16, E4M3])
def test_decode_attention_leaves_out_pages_outside_the_cache(store, page):
    cache, table, n, q, keys, values, _ = filled(3, [400, 200], 4, 2, 128, page, store)
    table[0, 1], table[0, 3], table[1, 0] = -1, cache.pages, 2 ** 31 - 1
    keep = [torch.ones(400, dtype=torch.bool), torch.ones(200, dtype=torch.bool)]
    keep[0][page: 2 * page] = keep[0][3 * page: 4 * page] = keep[1][:page] = False
    out, lse = tccl_amd.decode_attention(q.to(DEV), cache, table, n, return_lse=True)
    check_attention(out, lse, q, [k[m] for k, m in zip(keys, keep)], [v[m] for v, m in zip(values, keep)])
    table.fill_(-1)
    out, lse = tccl_amd.decode_attention(q.to(DEV), cache, table, n, return_lse=True)
    assert not out.any() and (lse == -math.inf).all()


def test_decode_attention_nan_in_a_live_token_reaches_its_heads_only():
    cache, table, n, q, keys, values, slots = filled(2, [100, 100], 4, 2, 64, 16, BF16)
    k, v = tccl_amd.cache_read(cache, slots[0][50:51].to(DEV))
    v[0, 1, 3] = math.nan
    tccl_amd.cache_write(cache, k, v, slots[0][50:51].to(DEV))
    out = tccl_amd.decode_attention(q.to(DEV), cache, table, n).cpu()
    bad = torch.isnan(out)
    assert bad[0, 2:, 3].all() and bad.sum() == 2
    k[0, 0, 0] = math.nan
    tccl_amd.cache_write(cache, k, torch.zeros_like(v), slots[0][50:51].to(DEV))
    out = tccl_amd.decode_attention(q.to(DEV), cache, table, n).cpu()
    bad = torch.isnan(out)
    assert bad[0, :2].all() and bad.sum() == 2 * 64


@pytest.mark.parametrize("store", [BF16, E4M3])
def test_decode_attention_of_sequences_that_share_pages(store):
    """A prefix in the cache once for all sequences, as a table row for all (a stride of 0) and as rows that part later; a length of
    2^31 - 1 is what the table has room for."""
    cache, table, n, q, keys, values, _ = filled(2, [700, 64, 130], 8, 2, 64, 16, store, seed=12)
    one = table[:1, :44].expand(3, 44)
    lengths = [700, 33, 2 ** 31 - 1]
    out, lse = tccl_amd.decode_attention(q.to(DEV), cache, one, torch.tensor(lengths, dtype=torch.int32, device=DEV), return_lse=True)
    have = [700, 33, 704]
    written = [torch.cat((x[0], torch.full((4, 2, 64), math.nan).double())) for x in (keys, values)]       # 4 tokens nobody wrote
    check_attention(out[:2], lse[:2], q[:2], [written[0][:m] for m in have[:2]], [written[1][:m] for m in have[:2]])
    assert torch.isnan(out[2]).all() and torch.isnan(lse[2]).all()
    mixed = table[:, :44].clone()
    mixed[1:, :4] = table[0, :4]
    mixed[2, 4:9] = table[2, :5]
    n = torch.tensor([700, 64, 64 + 80], dtype=torch.int32, device=DEV)
    out, lse = tccl_amd.decode_attention(q.to(DEV), cache, mixed, n, return_lse=True)
    held = [[x[0], x[0][:64], torch.cat((x[0][:64], x[2][:80]))] for x in (keys, values)]
    check_attention(out, lse, q, *held)


# ---------------------------------------------------------------- the join over ranks

@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("world,shape", [(1, (1, 64)), (2, (3, 5, 128)), (3, (17, 256)), (4, (1000, 64)), (5, (9, 64)), (6, (2, 2, 2, 128)),
                                          (7, (33, 128)), (8, (70_001, 64))])
def test_attention_all_reduce(world, shape, dtype):
    rng = torch.Generator().manual_seed(world)
    outs = [torch.randn(shape, generator=rng).to(dtype) for _ in range(world)]
    lses = [4 * torch.randn(shape[:-1], generator=rng) for _ in range(world)]
    for r in range(world):
        flat = lses[r].view(-1)
        flat[r::5] = -math.inf                                    # a rank without tokens, whose buffer holds anything
        outs[r].view(-1, shape[-1])[r::5] = math.nan
        flat[2::7] = -math.inf                                    # rows that no rank has tokens for
    for r in range(world):
        lses[r].view(-1)[3::11] -= 1e4
    o, l = world_of(outs), world_of(lses)
    got, lse = tccl_amd.attention_all_reduce(o.tensor(world - 1), l.tensor(world - 1))
    want, want_lse = ref.join(outs, lses)
    magnitude, _ = ref.join([x.double().abs() for x in outs], lses)
    # exp off by 4, `world` sums twice, a division and a product; the logarithm's argument is off by as much
    within(got, want, half_step(dtype) * want.abs() * (1 + 2.0 ** -7) + (2 * world + 12) * U * magnitude, "out")
    within(lse, want_lse, (world + 12) * U + 4 * U * torch.nan_to_num(want_lse.abs(), posinf=0.0), "lse")
    none, none_lse = tccl_amd.attention_all_reduce(o.tensor(0)[:0], l.tensor(0)[:0])
    assert none.numel() == 0 and none_lse.numel() == 0
    into = torch.empty_like(got)
    again, _ = tccl_amd.attention_all_reduce(o.tensor(0), l.tensor(0), out=into)
    assert again is into
    assert_bit_equal(again, got, "another rank's call")


def test_attention_all_reduce_behind_four_gib():
    rows, dim, some = 36_000_007, 64, 9                                 # 2.3e9 elements, 4.6e9 bytes
    rng = torch.Generator().manual_seed(18)
    o, l = tccl_amd.empty_world(2, (rows, dim), BF16, DEV), tccl_amd.empty_world(2, (rows,), F32, DEV)
    outs, lses = [torch.randn(some, dim, generator=rng).to(BF16) for _ in range(2)], [torch.randn(some, generator=rng) for _ in range(2)]
    for r in range(2):
        o.tensor(r).zero_()
        l.tensor(r).fill_(-math.inf)
        o.tensor(r)[-some:] = outs[r].to(DEV)
        l.tensor(r)[-some:] = lses[r].to(DEV)
    got, lse = tccl_amd.attention_all_reduce(o.tensor(0), l.tensor(0))
    want, want_lse = ref.join(outs, lses)
    magnitude, _ = ref.join([x.double().abs() for x in outs], lses)
    within(got[-some:], want, half_step(BF16) * want.abs() * (1 + 2.0 ** -7) + 16 * U * magnitude, "out")
    within(lse[-some:], want_lse, 14 * U + 4 * U * want_lse.abs(), "lse")
    assert not got[:-some].any() and (lse[:-some] == -math.inf).all()


def test_outputs_in_the_place_of_inputs():
    """attention_all_reduce into one of the ranks' buffers and decode_attention into its queries: the same bits as apart."""
    rng = torch.Generator().manual_seed(3)
    outs, lses = [torch.randn(5000, 64, generator=rng) for _ in range(3)], [torch.randn(5000, generator=rng) for _ in range(3)]
    o, l = world_of(outs), world_of(lses)
    want, want_lse = tccl_amd.attention_all_reduce(o.tensor(0), l.tensor(0))
    got, lse = tccl_amd.attention_all_reduce(o.tensor(0), l.tensor(0), out=o.tensor(1))
    assert got is o.tensor(1)
    assert_bit_equal(got, want, "in place")
    assert_bit_equal(lse, want_lse, "in place, lse")
    for lengths, heads in (([700, 3, 20011, 0], (6, 2)), ([40, 17], (70, 1))):            # split and not
        cache, table, n, q, *_ = filled(2, lengths, *heads, 64, 16, BF16, seed=4)
        queries = q.to(DEV)
        want, want_lse = tccl_amd.decode_attention(queries, cache, table, n, return_lse=True)
        got, lse = tccl_amd.decode_attention(queries, cache, table, n, out=queries, return_lse=True)
        assert got is queries
        assert_bit_equal(got, want, "in place of the queries")
        assert_bit_equal(lse, want_lse, "lse")


# ---------------------------------------------------------------- together, streams, graphs, per-rank programs

@pytest.mark.parametrize("store", [BF16, E4M3])
def test_a_serving_step_over_ranks(store):
    """Projections summed, normed and rotated; keys and values written to pages on all ranks; the new tokens' attention as one
    call over all ranks, and as one call per rank over its own pages joined by attention_all_reduce."""
    world, batch, q_heads, kv_heads, dim, page = 4, 3, 8, 2, 128, 16
    lengths = [70, 33, 129]
    heads = (q_heads, kv_heads, kv_heads)
    parts, w, _, inv_freq, _ = norm_inputs(world, sum(lengths), heads, dim, dim, BF16, seed=11)
    positions = torch.cat([torch.arange(n) for n in lengths])
    group = world_of(parts)
    q, k, v = tccl_amd.qk_norm_rope(group.tensor(0), w[0].to(DEV), w[1].to(DEV), positions.to(DEV), inv_freq.to(DEV), q_heads, kv_heads)
    cache = tccl_amd.PagedCache(world, 10, page, kv_heads, dim, dtype=store, device=DEV)
    # page j of a sequence lies on rank j % world
    width = 9
    table = torch.tensor([[(j % world) * 10 + b * 3 + j // world for j in range(width)] for b in range(batch)], dtype=torch.int32)
    slots = torch.cat([table[b].long()[torch.arange(n) // page] * page + torch.arange(n) % page for b, n in enumerate(lengths)])
    tccl_amd.cache_write(cache, k, v, slots.to(DEV))
    last = torch.tensor(lengths).cumsum(0) - 1
    newest = q[last.to(DEV)]
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    whole, whole_lse = tccl_amd.decode_attention(newest, cache, table.to(DEV), n, return_lse=True)
    held = [ref.stored(t.cpu(), store).split(lengths) for t in (k, v)]
    check_attention(whole, whole_lse, newest.cpu(), *held)

    outs = tccl_amd.empty_world(world, (batch, q_heads, dim), BF16, DEV)
    lses = tccl_amd.empty_world(world, (batch, q_heads), F32, DEV)
    for r in range(world):
        mine = table[:, r::world]
        have = torch.tensor([sum(min(page, max(0, length - j * page)) for j in range(r, width, world)) for length in lengths], dtype=torch.int32)
        tccl_amd.decode_attention(newest, cache, mine.to(DEV).contiguous(), have.to(DEV), out=outs.tensor(r), lse=lses.tensor(r))
    joined, joined_lse = tccl_amd.attention_all_reduce(outs.tensor(0), lses.tensor(0))
    want, want_lse = ref.attention(newest.cpu(), *held)
    magnitude, _ = ref.attention(newest.cpu(), held[0], [t.abs() for t in held[1]])
    # parts rounded to bf16, the joint once more: two half steps of the parts' magnitude and what check_attention allows
    within(joined, want, 2 * half_step(BF16) * magnitude * (1 + 2.0 ** -6) + 2.0 ** -12 * magnitude, "joined")
    within(joined_lse, want_lse, 2.0 ** -14 * (1 + want_lse.abs()), "joined lse")


def test_on_another_stream_and_two_at_once():
    a = filled(2, [3000, 100], 8, 2, 128, 16, BF16, seed=1)
    b = filled(3, [2500, 900], 8, 2, 128, 16, E4M3, seed=2)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s, (cache, table, n, q, *_rest) in zip(streams, (a, b)):
            queries = q.to(DEV)
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(tccl_amd.decode_attention(queries, cache, table, n, return_lse=True))
                queries.record_stream(s)
    torch.cuda.synchronize()
    for i, (out, lse) in enumerate(got):
        _, _, _, q, keys, values, _ = (a, b)[i % 2]
        check_attention(out, lse, q, keys, values)


@pytest.mark.parametrize("call", ["write", "read", "attention"])
def test_a_cache_dropped_while_another_stream_uses_it(call):
    """The buffers are not handed out again before that stream has passed the call."""
    cache, table, n, q, keys, values, slots = filled(2, [700, 100], 8, 2, 128, 16, BF16, seed=1)
    at, queries = torch.cat(slots).to(DEV), q.to(DEV)
    k, v = (torch.cat(x).to(BF16).to(DEV) for x in (keys, values))
    nbytes, pointers = cache.group.tensors[0].numel(), set(cache.group.buffer_ptrs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        if call == "write":
            tccl_amd.cache_write(cache, k, v, at)
        elif call == "read":
            got = tccl_amd.cache_read(cache, at)
        else:
            out = tccl_amd.decode_attention(queries, cache, table, n)
    del cache
    others = [torch.full((nbytes,), 0xFF, dtype=torch.uint8, device=DEV) for _ in range(2)]
    assert not side.query(), "the side stream was to be busy still"
    assert pointers.isdisjoint(t.data_ptr() for t in others)
    torch.cuda.synchronize()
    if call == "write":
        assert all((t == 0xFF).all() for t in others)
    elif call == "read":
        assert torch.equal(got[0], k) and torch.equal(got[1], v)
    else:
        check_attention(out, None, q, keys, values)


def captured(fn):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = fn()
    return graph, result


def test_a_decode_step_in_two_graphs():
    """A whole step captured twice over different batches and replayed alternately with new inputs, beside eager calls."""
    world, q_heads, kv_heads, dim, page = 2, 8, 2, 64, 16
    heads = (q_heads, kv_heads, kv_heads)
    steps = []
    for seed, lengths in ((1, [900, 5]), (2, [3, 1200])):
        cache, table, n, *_ = filled(world, lengths, q_heads, kv_heads, dim, page, E4M3, seed=seed)
        parts, w, positions, inv_freq, grads = norm_inputs(world, 2, heads, dim, dim, BF16, seed=seed)
        group = world_of(parts)
        dw, pos, inv = [t.to(DEV) for t in w], positions.to(DEV), inv_freq.to(DEV)
        where = torch.stack([table[b, (m - 1) // page].long() * page + (m - 1) % page for b, m in enumerate(lengths)])
        dy = [g.to(DEV) for g in grads]

        def step(group=group, dw=dw, pos=pos, inv=inv, cache=cache, table=table, n=n, where=where, dy=dy):
            q, k, v = tccl_amd.qk_norm_rope(group.tensor(0), *dw, pos, inv, q_heads, kv_heads)
            tccl_amd.cache_write(cache, k, v, where)
            out, lse = tccl_amd.decode_attention(q, cache, table, n, return_lse=True)
            return (out, lse, *tccl_amd.cache_read(cache, where), *tccl_amd.qk_norm_rope_backward(*dy, group.tensor(0), *dw, pos, inv))

        steps.append((step, group, *captured(step)))
    rng = torch.Generator(device=DEV).manual_seed(0)
    for turn in range(5):
        for step, group, _, _ in steps:
            for t in group.tensors:
                t.copy_(torch.randn(t.shape, generator=rng, device=DEV))
        steps[turn % 2][2].replay()
        steps[1 - turn % 2][2].replay()
        torch.cuda.synchronize()
        for step, _, _, result in steps:
            kept = [t.clone() for t in result]
            for got, want in zip(kept, step()):
                assert_bit_equal(got, want, f"replay {turn}")


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_parts_and_their_join_in_a_graph(dtype):
    """Each rank's attention over its own pages into symmetric buffers and their join, captured and replayed over new queries."""
    world, lengths = 3, [900, 40, 0]
    parts = [filled(1, lengths, 8, 2, 64, 16, BF16, seed=20 + r) for r in range(world)]
    q = parts[0][3].to(DEV)
    outs = tccl_amd.empty_world(world, (3, 8, 64), BF16, DEV)
    lses = tccl_amd.empty_world(world, (3, 8), F32, DEV)
    wide = tccl_amd.empty_world(world, (3, 8, 64), dtype, DEV)

    def step():
        for r, (cache, table, n, *_) in enumerate(parts):
            tccl_amd.decode_attention(q, cache, table, n, out=outs.tensor(r), lse=lses.tensor(r))
            wide.tensor(r).copy_(outs.tensor(r))
        return tccl_amd.attention_all_reduce(wide.tensor(1), lses.tensor(1))

    graph, result = captured(step)
    rng = torch.Generator(device=DEV).manual_seed(1)
    for turn in range(4):
        q.copy_(torch.randn(q.shape, generator=rng, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in result]
        for got, want in zip(kept, step()):
            assert_bit_equal(got, want, f"replay {turn}")
        keys = [torch.cat([p[4][b] for p in parts]) for b in range(3)]
        values = [torch.cat([p[5][b] for p in parts]) for b in range(3)]
        want, want_lse = ref.attention(q.cpu(), keys, values)
        magnitude, _ = ref.attention(q.cpu(), keys, [v.abs() for v in values])
        # as in test_a_serving_step_over_ranks: the parts' rounding to bf16, the joint's, and what the parts are off by
        within(kept[0], want, 2 * half_step(BF16) * magnitude * (1 + 2.0 ** -6) + 2.0 ** -12 * magnitude, "joined")
        within(kept[1], want_lse, 2.0 ** -14 * (1 + torch.nan_to_num(want_lse.abs(), posinf=0.0)), "joined lse")


def test_in_a_per_rank_program():
    world, heads, dim, tokens = 4, (4, 2, 2), 64, 6
    parts, w, positions, inv_freq, _ = norm_inputs(world, tokens, heads, dim, dim, BF16, seed=21)
    dw = [t.to(DEV) for t in w]
    cache = tccl_amd.PagedCache(world, 2, 16, 2, dim, device=DEV)
    table = torch.tensor([[0, 2]], dtype=torch.int32, device=DEV)

    def main(rank, world_size):
        t = tccl_amd.spmd.empty_strided_p2p(parts[0].shape, None, BF16, DEV)
        t.copy_(parts[rank])
        q, k, v = tccl_amd.qk_norm_rope(t, *dw, positions.to(DEV), inv_freq.to(DEV), 4, 2)
        if rank == 2:
            tccl_amd.cache_write(cache, k, v, torch.arange(tokens, device=DEV))
        out = tccl_amd.decode_attention(q[-1:], cache, table, torch.tensor([tokens], dtype=torch.int32, device=DEV))
        o = tccl_amd.spmd.empty_strided_p2p(out.shape, None, BF16, DEV)
        l = tccl_amd.spmd.empty_strided_p2p(out.shape[:-1], None, F32, DEV)
        o.copy_(out)
        l.fill_(0.5)
        joined, _ = tccl_amd.attention_all_reduce(o, l)
        return q.cpu(), k.cpu(), v.cpu(), out.cpu(), joined.cpu()

    results = tccl_amd.spmd.run(world, main)
    q, k, v = results[0][:3]
    check_forward((q, k, v), parts, w, positions, inv_freq, heads, 1e-6, False)
    check_attention(results[0][3], None, q[-1:], [k.double()], [v.double()])
    for r in results:
        for a, b in zip(r[:4], results[0][:4]):
            assert_bit_equal(a, b, "every rank has the same")
        # equal weights over equal parts: the parts themselves, up to the fp32 division by the number of ranks
        within(r[4], r[3].double(), half_step(BF16) * r[3].double().abs() * 1.01, "joined")


def test_caches_of_the_ranks_own_in_a_per_rank_program():
    """Each rank makes a cache for its part of the tokens, attends to it, and the parts are joined."""
    world, lengths, page = 3, [70, 5, 0], 16
    rng = torch.Generator().manual_seed(22)
    q = torch.randn(3, 4, 64, generator=rng).to(BF16)
    k, v = ([torch.randn(world, n, 2, 64, generator=rng).to(BF16) for n in lengths] for _ in range(2))
    table = torch.arange(15, dtype=torch.int32).view(3, 5)

    def main(rank, world_size):
        cache = tccl_amd.PagedCache(1, 15, page, 2, 64, device=DEV)
        slots = torch.cat([b * 5 * page + torch.arange(n) for b, n in enumerate(lengths)])
        tccl_amd.cache_write(cache, *(torch.cat([t[rank] for t in x]).to(DEV) for x in (k, v)), slots.to(DEV))
        out = tccl_amd.spmd.empty_strided_p2p((3, 4, 64), None, BF16, DEV)
        lse = tccl_amd.spmd.empty_strided_p2p((3, 4), None, F32, DEV)
        tccl_amd.decode_attention(q.to(DEV), cache, table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), out=out, lse=lse)
        joined, joined_lse = tccl_amd.attention_all_reduce(out, lse)
        return joined.cpu(), joined_lse.cpu()

    results = tccl_amd.spmd.run(world, main)
    keys, values = ([t.flatten(0, 1).double() for t in x] for x in (k, v))
    want, want_lse = ref.attention(q, keys, values)
    magnitude, _ = ref.attention(q, keys, [t.abs() for t in values])
    for joined, joined_lse in results:
        # as in test_a_serving_step_over_ranks
        within(joined, want, 2 * half_step(BF16) * magnitude * (1 + 2.0 ** -6) + 2.0 ** -12 * magnitude, "joined")
        within(joined_lse, want_lse, 2.0 ** -14 * (1 + torch.nan_to_num(want_lse.abs(), posinf=0.0)), "joined lse")

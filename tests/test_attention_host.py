"""The attention operators on a machine without a GPU: what their entry points and host wrappers refuse before
anything is launched, the struct that crosses the ABI, and the 64-bit reference against differences."""
import ctypes
import gc
import math
import os
import shutil
import subprocess
import weakref

import pytest
import torch

import tccl_amd
from oracle import attention_ref as ref
from tccl_amd import _lib, attention

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, EINVAL, EALIGN, ESCRATCH = _lib.TCCL_OK, _lib.TCCL_EINVAL, _lib.TCCL_EALIGN, _lib.TCCL_ESCRATCH


def desc(**kw):
    d = _lib.PagedCacheDesc()
    d.world, d.pages_per_rank, d.page_size, d.kv_heads, d.head_dim, d.dtype = 2, 3, 16, 4, 64, _lib.TCCL_BF16
    d.bufs[0], d.bufs[1] = 0x10000, 0x20000
    for k, v in kw.items():
        if k == "bufs":
            d.bufs[1] = v
        else:
            setattr(d, k, v)
    return ctypes.byref(d)


def test_norm_entry_points_check_their_arguments():
    lib = tccl_amd.load_library()
    good = dict(bufs=_lib.ptr_array([0x1000, 0x2000]), world=2, q=0x3000, k=0x4000, v=0x5000, qw=0x6000, kw=0x7000,
                pos=0x8000, inv=0x9000, tokens=0, heads=(4, 2, 2), dim=64, rotary=64, inter=0, eps=1e-6, dtype=0)

    def fwd(**kw):
        c = {**good, **kw}
        return lib.tccl_qk_norm_rope(c["bufs"], c["world"], c["q"], c["k"], c["v"], c["qw"], c["kw"], c["pos"], c["inv"],
                                     c["tokens"], *c["heads"], c["dim"], c["rotary"], c["inter"], c["eps"], c["dtype"], None)

    def bwd(ws=0x100000, nbytes=1 << 24, dqw=0xA000, **kw):
        c = {**good, "tokens": 8, **kw}
        return lib.tccl_qk_norm_rope_backward(c["bufs"], c["world"], c["q"], c["k"], c["v"], c["qw"], c["kw"], c["pos"], c["inv"],
                                              0xC000, dqw, 0xB000, ws, nbytes, c["tokens"], *c["heads"], c["dim"],
                                              c["rotary"], c["inter"], c["eps"], c["dtype"], None)

    assert fwd() == OK                                        # no tokens: nothing to launch
    bad = [dict(bufs=None), dict(world=0), dict(world=9), dict(bufs=_lib.ptr_array([0x1000, None])), dict(q=None), dict(k=None),
           dict(v=None), dict(qw=None), dict(kw=None), dict(pos=None), dict(inv=None), dict(dim=96), dict(rotary=8),
           dict(rotary=80), dict(rotary=-16), dict(heads=(0, 0, 0)), dict(heads=(-1, 2, 2)), dict(eps=-1.0),
           dict(eps=math.nan), dict(dtype=2), dict(dtype=7), dict(tokens=1 << 31)]
    assert fwd(tokens=1 << 24) == EINVAL                      # more workgroups than one launch has
    for kw in bad:
        assert fwd(**kw) == EINVAL, kw
        assert bwd(**kw) == EINVAL, kw
    for kw in (dict(bufs=_lib.ptr_array([0x1000, 0x2008])), dict(q=0x3008), dict(kw=0x7004), dict(v=0x5002)):
        assert fwd(**kw) == EALIGN, kw
        assert bwd(**kw) == EALIGN, kw
    assert fwd(heads=(4, 2, 0), v=None) == OK                 # no value heads: no output for them
    assert fwd(rotary=0, inv=None) == OK
    assert bwd(ws=None) == EINVAL and bwd(dqw=None) == EINVAL
    assert bwd(ws=0x100004) == EALIGN and bwd(dqw=0xA004) == EALIGN
    need = lib.tccl_qk_norm_rope_backward_workspace(64)
    assert need > 0 and lib.tccl_qk_norm_rope_backward_workspace(96) == 0
    assert bwd(nbytes=need - 1) == ESCRATCH


def test_cache_entry_points_check_their_arguments():
    lib = tccl_amd.load_library()
    assert lib.tccl_paged_cache_bytes(desc()) == 3 * 4 * 16 * 64 * 2 * 2
    assert lib.tccl_paged_cache_bytes(desc(dtype=_lib.TCCL_E4M3)) == 3 * 4 * 16 * (64 * 2 + 2)
    shapes = [dict(world=0), dict(world=9), dict(pages_per_rank=0), dict(pages_per_rank=1 << 30, world=3), dict(page_size=8),
              dict(page_size=48), dict(page_size=512), dict(kv_heads=0), dict(kv_heads=65536), dict(head_dim=80), dict(dtype=1)]

    def write(d, k=0x1000, v=0x2000, strides=(256, 64, 256, 64), slots=0x3000, tokens=0, dtype=0):
        return lib.tccl_cache_write(d, k, v, *strides, slots, tokens, dtype, None)

    def read(d, slots=0x3000, tokens=0, k=0x1000, v=0x2000, dtype=0):
        return lib.tccl_cache_read(d, slots, tokens, k, v, dtype, None)

    for kw in shapes:
        assert lib.tccl_paged_cache_bytes(desc(**kw)) == 0, kw
        assert write(desc(**kw)) == EINVAL and read(desc(**kw)) == EINVAL, kw
    assert lib.tccl_paged_cache_bytes(None) == 0 and write(None) == EINVAL and read(None) == EINVAL
    assert write(desc(bufs=None)) == EINVAL and read(desc(bufs=None)) == EINVAL
    assert write(desc(bufs=0x20008)) == EALIGN and read(desc(bufs=0x20008)) == EALIGN
    assert write(desc()) == OK and read(desc()) == OK
    for kw in (dict(k=None), dict(v=None), dict(slots=None), dict(dtype=2), dict(tokens=(1 << 29) + 1)):
        assert write(desc(), **kw) == EINVAL and read(desc(), **kw) == EINVAL, kw
    assert write(desc(), k=0x1008) == EALIGN and read(desc(), v=0x2004) == EALIGN
    assert write(desc(), strides=(256, 60, 256, 64)) == EALIGN and write(desc(), strides=(256, 64, 257, 64)) == EALIGN


def test_attention_entry_points_check_their_arguments():
    lib = tccl_amd.load_library()

    def attn(d, q=0x1000, strides=(512, 64), table=0x2000, lengths=0x3000, out=0x4000, lse=0x5000, ws=None, nbytes=0, batch=0,
             heads=8, most=64):
        return lib.tccl_decode_attention(d, q, *strides, table, 4, lengths, out, lse, ws, nbytes, batch, heads, most, 0.1, None)

    assert attn(desc()) == OK
    assert attn(desc(), lse=None) == OK                       # no lse wanted
    assert attn(desc(), table=None, most=0) == OK             # no sequence can have a token
    for kw in (dict(q=None), dict(lengths=None), dict(out=None), dict(table=None), dict(heads=6), dict(heads=0), dict(most=-1), dict(most=(1 << 30) + 1),
               dict(batch=(1 << 20) + 1)):
        assert attn(desc(), **kw) == EINVAL, kw
    assert attn(desc(page_size=20)) == EINVAL and attn(None) == EINVAL
    for kw in (dict(q=0x1008), dict(out=0x4008), dict(ws=0x6004), dict(strides=(512, 60)), dict(strides=(508, 64))):
        assert attn(desc(), **kw) == EALIGN, kw
    assert attn(desc(), batch=5000, heads=8192, most=64) == EINVAL               # more workgroups than one launch has
    sizes = [lib.tccl_decode_attention_workspace(n, 8, 4, 64, 3000) for n in (1, 100, 4096, 4097, 9000)]
    assert sizes[3] >= max(sizes[:3]) and sizes[4] == sizes[3] == sizes[2]        # launches of 4,096 share it
    need = lib.tccl_decode_attention_workspace(1, 8, 4, 64, 100_000)
    assert need > 0
    assert attn(desc(), batch=1, most=100_000) == ESCRATCH
    assert attn(desc(), batch=1, most=100_000, ws=0x10000, nbytes=need - 1) == ESCRATCH
    assert lib.tccl_decode_attention_workspace(1, 6, 4, 64, 100) == 0

    two, odd, null = _lib.ptr_array([0x1000, 0x2000]), _lib.ptr_array([0x1000, 0x2008]), _lib.ptr_array([0x1000, None])

    def join(outs=two, lses=two, world=2, out=0x3000, lse=0x4000, rows=0, dim=64, dtype=0):
        return lib.tccl_attention_all_reduce(outs, lses, world, out, lse, rows, dim, dtype, None)

    assert join() == OK
    for kw in (dict(outs=None), dict(lses=None), dict(outs=null), dict(lses=null), dict(world=0), dict(world=9), dict(out=None),
               dict(lse=None), dict(dim=80), dict(dtype=2)):
        assert join(**kw) == EINVAL, kw
    for kw in (dict(outs=odd), dict(lses=odd), dict(out=0x3004), dict(lse=0x4004)):
        assert join(**kw) == EALIGN, kw


def test_cache_struct_matches_the_header(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    src = tmp_path / "layout.c"
    names = [f[0] for f in _lib.PagedCacheDesc._fields_]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "tccl_amd.h"\nint main(void) {\n  printf("%zu", sizeof(tccl_paged_cache));\n'
                   + "".join(f'  printf(" %zu", offsetof(tccl_paged_cache, {n}));\n' for n in names)
                   + '  printf(" %d\\n", TCCL_E4M3);\n  return 0;\n}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    c = _lib.PagedCacheDesc
    assert got == [ctypes.sizeof(c), *(getattr(c, n).offset for n in names), _lib.TCCL_E4M3]


# ---------------------------------------------------------------- the Python wrappers' refusals (CPU tensors)

def projection(tokens=4, columns=8 * 64, dtype=torch.bfloat16):
    return tccl_amd.empty_world(2, (tokens, columns), dtype, device="cpu")


def norm(x, qw=None, kw=None, positions=None, inv_freq=None, q_heads=4, k_heads=2, **kwargs):
    tokens = x.shape[0]
    w = torch.ones(64, dtype=x.dtype)
    return tccl_amd.qk_norm_rope(x, w if qw is None else qw, w if kw is None else kw,
                                 torch.arange(tokens) if positions is None else positions,
                                 torch.ones(32, dtype=torch.float64) if inv_freq is None else inv_freq, q_heads, k_heads, **kwargs)


def test_qk_norm_rope_refusals():
    x = projection().tensor(0)
    cases = [dict(qw=torch.ones(80, dtype=x.dtype)), dict(kw=torch.ones(64)), dict(kw=torch.ones(128, dtype=x.dtype)),
             dict(qw=torch.ones(128, dtype=x.dtype)[::2]), dict(positions=torch.arange(4).int()), dict(positions=torch.arange(5)),
             dict(positions=torch.arange(8)[::2]), dict(inv_freq=torch.ones(32)), dict(inv_freq=torch.ones(12, dtype=torch.float64)),
             dict(inv_freq=torch.ones(40, dtype=torch.float64)), dict(inv_freq=torch.ones(4, 8, dtype=torch.float64)),
             dict(q_heads=7), dict(q_heads=-1), dict(k_heads=-2)]
    for kw in cases:
        with pytest.raises(ValueError):
            norm(x, **kw)
    with pytest.raises(AssertionError, match="bfloat16"):
        norm(projection(dtype=torch.float16).tensor(0))
    with pytest.raises(ValueError, match="columns"):
        norm(x.view(-1)[:7 * 72].view(7, 72))
    with pytest.raises(RuntimeError, match="symmetric group"):
        norm(torch.zeros(4, 8 * 64, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="first element"):
        norm(x[1:])
    with pytest.raises(ValueError, match="GPU"):
        norm(x)


def test_qk_norm_rope_backward_refusals():
    x = projection().tensor(0)
    w = torch.ones(64, dtype=x.dtype)
    rest = (w, w, torch.arange(4), torch.ones(32, dtype=torch.float64))
    g = [torch.zeros(4, n, 64, dtype=x.dtype) for n in (4, 2, 2)]
    for bad in (torch.zeros(4, 3, 64, dtype=x.dtype), torch.zeros(4, 4, 64), torch.zeros(5, 4, 64, dtype=x.dtype),
                torch.zeros(4, 256, dtype=x.dtype), torch.zeros(4, 64, 4, dtype=x.dtype).transpose(1, 2)):
        with pytest.raises(ValueError):
            tccl_amd.qk_norm_rope_backward(bad, g[1], g[2], x, *rest)
    with pytest.raises(ValueError, match="GPU"):
        tccl_amd.qk_norm_rope_backward(*g, x, *rest)


def test_paged_cache_refusals():
    good = dict(world_size=2, pages_per_rank=3, page_size=16, kv_heads=2, head_dim=64, device="cpu")
    for kw in (dict(world_size=0), dict(world_size=9), dict(pages_per_rank=0), dict(page_size=24), dict(page_size=8), dict(kv_heads=0),
               dict(head_dim=96), dict(dtype=torch.float32), dict(pages_per_rank=1 << 30)):
        with pytest.raises(ValueError):
            tccl_amd.PagedCache(**{**good, **kw})
    cache = tccl_amd.PagedCache(**good)
    assert cache.pages == 6 and cache.slots == 96
    gone = weakref.ref(cache.group.tensors[1])
    gc.disable()
    try:
        cache = tccl_amd.PagedCache(**good)
        assert gone() is None, "a dropped cache keeps its buffers until a garbage collection"
    finally:
        gc.enable()
    k, slots = torch.zeros(5, 2, 64), torch.arange(5)
    for bad in ((k[:4], k, slots), (k, k[:, :1], slots), (k, k.bfloat16(), slots), (k, k, slots.int()), (k, k, torch.arange(10)[::2]),
                (k.transpose(1, 2).contiguous().transpose(1, 2), k, slots), (torch.zeros(5, 2, 65)[..., :64], k, slots),
                (torch.zeros(641)[1:].view(5, 2, 64), k, slots)):
        with pytest.raises(ValueError):
            tccl_amd.cache_write(cache, *bad)
    with pytest.raises(AssertionError):
        tccl_amd.cache_write(cache, k.half(), k.half(), slots)
    with pytest.raises(ValueError, match="GPU"):
        tccl_amd.cache_write(cache, k, k, slots)
    with pytest.raises(ValueError):
        tccl_amd.cache_read(cache, slots.int())
    with pytest.raises(ValueError):
        tccl_amd.cache_read(cache, slots, dtype=torch.float16)
    with pytest.raises(ValueError):
        tccl_amd.cache_read(cache, slots, out=(k, k))                       # float32 where bfloat16 is asked for
    with pytest.raises(ValueError):
        tccl_amd.cache_read(cache, slots, dtype=torch.float32, out=(torch.zeros(641)[1:].view(5, 2, 64), k))
    with pytest.raises(ValueError, match="GPU"):
        tccl_amd.cache_read(cache, slots)


def test_a_cache_larger_than_an_address_space_is_refused():
    """40,000 heads of 256 x 2 x 256 bf16: 2^64 bytes and 5.9 GB more, of which 64 bits would hold the 5.9 GB."""
    lib = tccl_amd.load_library()
    pages, heads = -(-(1 << 46) // 40_000), 40_000
    assert pages * heads << 18 > 1 << 64 and pages < 1 << 31
    big = dict(pages_per_rank=pages, kv_heads=heads, page_size=256, head_dim=256, world=1)
    assert lib.tccl_paged_cache_bytes(desc(**big)) == 0
    assert lib.tccl_cache_write(desc(**big), 0x1000, 0x2000, 256, 256, 256, 256, 0x3000, 0, 0, None) == EINVAL
    assert lib.tccl_cache_read(desc(**big), 0x3000, 0, 0x1000, 0x2000, 0, None) == EINVAL
    assert lib.tccl_decode_attention(desc(**big), 0x1000, 512, 256, 0x2000, 4, 0x3000, 0x4000, None, None, 0, 0, heads, 64, 0.1, None) == EINVAL
    with pytest.raises(ValueError, match="bytes"):
        tccl_amd.PagedCache(1, pages, 256, heads, 256, device="cpu")
    half = dict(big, pages_per_rank=pages // 2 - 1)
    assert lib.tccl_paged_cache_bytes(desc(**half)) == half["pages_per_rank"] * heads << 18


def test_a_cache_tells_the_allocator_of_other_streams_once(monkeypatch):
    """So that a dropped cache's buffers stay its own until work on those streams is done."""
    cache = tccl_amd.PagedCache(2, 3, 16, 2, 64, device="cpu")
    told = []

    class Buffer:
        def record_stream(self, stream):
            told.append((self, stream))

    buffers = cache.group.tensors = [Buffer(), Buffer()]
    cache._streams = {None}                                            # made on the default stream
    state = {"raw": None, "capturing": False}
    monkeypatch.setattr(attention, "_stream", lambda device: ctypes.c_void_p(state["raw"]))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: f"stream {state['raw']}")

    def launch(raw, capturing=False):
        state.update(raw=raw, capturing=capturing)
        del told[:]
        assert cache._launch_stream().value == raw
        return told

    assert launch(None) == []
    assert launch(7, capturing=True) == []                             # nothing runs
    assert launch(7) == [(buffers[0], "stream 7"), (buffers[1], "stream 7")]
    assert launch(7) == [] and launch(None) == []
    assert len(launch(8)) == 2 and launch(7) == []


def test_decode_attention_refusals():
    cache = tccl_amd.PagedCache(2, 3, 16, 2, 64, device="cpu")
    q, table, lengths = torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for bad in ((q.float(), table, lengths), (q[:2], table, lengths), (q[:, :3], table, lengths), (q[..., :32], table, lengths),
                (q, table.long(), lengths), (q, table[:2], lengths), (q, table, lengths.long()), (q, table, lengths[None]),
                (q, torch.zeros(3, 4, dtype=torch.int32)[:, ::2], lengths), (q.transpose(1, 2).contiguous().transpose(1, 2), table, lengths)):
        with pytest.raises(ValueError):
            tccl_amd.decode_attention(bad[0], cache, *bad[1:])
    for kw in (dict(max_length=-1), dict(out=q.float()), dict(out=torch.zeros(3, 4, 32, dtype=torch.bfloat16)), dict(lse=torch.zeros(3, 3)),
               dict(lse=torch.zeros(3, 4, dtype=torch.float64))):
        with pytest.raises(ValueError):
            tccl_amd.decode_attention(q, cache, table, lengths, **kw)
    with pytest.raises(ValueError, match="GPU"):
        tccl_amd.decode_attention(q, cache, table, lengths)


def test_attention_all_reduce_refusals():
    outs, lses = tccl_amd.empty_world(2, (6, 64), torch.float32, "cpu"), tccl_amd.empty_world(2, (6,), torch.float32, "cpu")
    other = tccl_amd.empty_world(3, (6,), torch.float32, "cpu")
    o, l = outs.tensor(0), lses.tensor(0)
    for bad in ((o, lses.tensor(1)), (o, other.tensor(0)), (o, l[:5]), (o, l.view(6, 1)), (o.view(12, 32), l)):
        with pytest.raises(ValueError):
            tccl_amd.attention_all_reduce(*bad)
    with pytest.raises(RuntimeError):
        tccl_amd.attention_all_reduce(torch.zeros(6, 64), l)
    with pytest.raises(RuntimeError):
        tccl_amd.attention_all_reduce(o, torch.zeros(6))
    with pytest.raises(AssertionError):
        tccl_amd.attention_all_reduce(o.half(), l)
    with pytest.raises(ValueError, match="out must be"):
        tccl_amd.attention_all_reduce(o, l, out=torch.zeros(6, 128))
    with pytest.raises(ValueError, match="GPU"):
        tccl_amd.attention_all_reduce(o, l)


@pytest.mark.parametrize("which", [0, 1])
def test_attention_all_reduce_looks_at_both_groups_expired_waits(which, monkeypatch):
    """Outputs or softmax sums that a collective left half reduced are not joined unnoticed."""
    groups = [tccl_amd.empty_world(2, (6, 64), torch.float32, "cpu"), tccl_amd.empty_world(2, (6,), torch.float32, "cpu")]

    def expired():
        raise _lib.TcclError("a signalling collective", _lib.TCCL_ETIMEOUT, "a wait expired")

    monkeypatch.setattr(groups[which], "check_signals", expired)
    with pytest.raises(_lib.TcclError, match="wait expired"):
        tccl_amd.attention_all_reduce(groups[0].tensor(0), groups[1].tensor(0))


def test_attention_all_reduce_refuses_outputs_that_other_reads_would_meet():
    """A launch reads every rank's rows: an output over them is right row by row only, and not where each rank launches its own."""
    outs, lses = tccl_amd.empty_world(2, (8, 64), torch.float32, "cpu"), tccl_amd.empty_world(2, (8,), torch.float32, "cpu")
    o, l = outs.tensor(0)[:4], lses.tensor(0)[:4]
    for out in (outs.tensor(0)[1:5], outs.tensor(1)[3:7]):
        with pytest.raises(ValueError, match="overlap"):
            tccl_amd.attention_all_reduce(o, l, out=out)
    for out in (o, outs.tensor(1)[:4], outs.tensor(0)[4:], torch.zeros(4, 64)):     # in place, or apart: only the GPU is missing
        with pytest.raises(ValueError, match="GPU"):
            tccl_amd.attention_all_reduce(o, l, out=out)
    few, sums = tccl_amd.empty_world(2, (1, 64), torch.float32, "cpu"), tccl_amd.empty_world(2, (256,), torch.float32, "cpu")
    with pytest.raises(ValueError, match="overlap"):
        tccl_amd.attention_all_reduce(few.tensor(0), sums.tensor(0)[:1], out=sums.tensor(1)[:64].view(1, 64))

    def main(rank, world_size, peer):
        t = tccl_amd.spmd.empty_strided_p2p((8, 64), None, torch.float32, "cpu")
        s = tccl_amd.spmd.empty_strided_p2p((8,), None, torch.float32, "cpu")
        tccl_amd.attention_all_reduce(t, s, out=t if peer is None else outs.tensor(0))

    with pytest.raises(ValueError, match="overlap"):
        tccl_amd.spmd.run(2, main, None)
    with pytest.raises(ValueError, match="GPU"):
        tccl_amd.spmd.run(2, main, 1)


def test_groups_of_other_processes_are_refused():
    """The kernels read every rank's buffer without the in-kernel barrier that ranks in processes of their own need."""
    own = torch.zeros(4, 8 * 64, dtype=torch.bfloat16)
    tccl_amd.symm.register_remote(own, 0, [own.data_ptr(), own.data_ptr() + (1 << 20)])
    with pytest.raises(RuntimeError, match="other processes|other ranks"):
        norm(own)


# ---------------------------------------------------------------- the reference itself

@pytest.mark.parametrize("interleaved", [False, True])
def test_reference_gradients_against_differences(interleaved):
    torch.manual_seed(3)
    parts = [torch.randn(3, 4 * 64, dtype=torch.float64) for _ in range(2)]
    grads = [torch.randn(3, n, 64, dtype=torch.float64) for n in (2, 1, 1)]
    w = [torch.rand(64, dtype=torch.float64) + 0.5 for _ in range(2)]
    positions, inv_freq = torch.tensor([0, 7, 1000]), torch.rand(16, dtype=torch.float64)
    dx, dqw, dkw = ref.qk_norm_rope_grad(parts, grads, *w, positions, inv_freq, 1e-6, interleaved)

    def value(x, qw, kw):
        y = ref.qk_norm_rope(x, qw, kw, positions, inv_freq, 2, 1, 1e-6, interleaved)
        return sum((a * g).sum() for a, g in zip(y, grads))

    x, h = sum(parts), 1e-5
    for which, (at, got) in enumerate(((x, dx), (w[0], dqw), (w[1], dkw))):
        d = torch.randn_like(at)
        args = [[x, *w], [x, *w]]
        args[0][which], args[1][which] = at + h * d, at - h * d
        numeric = (value(*args[0]) - value(*args[1])) / (2 * h)
        # the third-order term h^2 |d|^3 f''' is about 1e-10 * 64; rounding 1e-16 |f| / h about 1e-10
        assert abs(numeric - (got * d).sum()) <= 1e-7 * (1 + (got * d).abs().sum())


def test_reference_storage():
    assert torch.equal(ref.stored(torch.tensor([[448.0, 1.0, 0.0, -448.0]]), torch.float8_e4m3fn), torch.tensor([[448.0, 1.0, 0.0, -448.0]], dtype=torch.float64))
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    codes = codes[torch.isfinite(codes)]
    assert torch.equal(ref.stored(codes[None], torch.float8_e4m3fn)[0], codes.double())      # every value is kept as it is
    y = torch.randn(64, 128)
    same = torch.ldexp((torch.ldexp(y, -_exponent(y))).to(torch.float8_e4m3fn).float(), _exponent(y))
    assert torch.equal(ref.stored(y, torch.float8_e4m3fn), same.double())


def _exponent(y):
    m, e = torch.frexp(y.abs().amax(-1, keepdim=True))
    return e - 9 + (m > 0.875).int()


def test_reference_storage_of_the_largest_rows():
    """Multiples of 2^120 stop at 240: a finite value is kept as a finite one, off by at most half a step of a code, 2^-4 of it."""
    x = torch.tensor([1.75, 1.9374, 1.9375, -1.9375, 2 - 2.0 ** -23], dtype=torch.float64)[:, None] * 2.0 ** 127
    got = ref.stored(x, torch.float8_e4m3fn)
    assert torch.equal(got[:, 0] / 2.0 ** 120, torch.tensor([224.0, 240.0, 240.0, -240.0, 240.0], dtype=torch.float64))
    assert torch.isfinite(got.to(torch.bfloat16)).all() and torch.isfinite(got.float()).all()
    assert ((got - x).abs() <= 2.0 ** -4 * x.abs()).all()

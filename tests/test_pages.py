"""CPU: argument checks of the operators over 8-bit caches and pages (C ABI and Python), and pins of their oracle."""

import ctypes
import math

import pytest
import torch

from kvskip_amd import _native, ext
from kvskip_amd import kvskip as K
from kvskip_amd._native import AttnArgs, Cache8Args, PageArgs, WriteArgs
from oracle import pages as OPG


def test_struct_layouts():
    lib = _native.lib()
    assert [lib.kvskip_struct_size(i) for i in (5, 6, 7)] == [ctypes.sizeof(x) for x in (Cache8Args, PageArgs, WriteArgs)]


def _attn(**kw):
    a = AttnArgs()
    a.q, a.k, a.v = 0x1000, 0x2000, 0x3000
    a.q_sb, a.q_sh = 32 * 128, 128
    a.k_sb, a.k_sh, a.k_st = 8 * 4096 * 128, 4096 * 128, 128
    a.v_sb, a.v_sh, a.v_st = a.k_sb, a.k_sh, a.k_st
    a.B, a.Hq, a.Hkv, a.T, a.D = 1, 32, 8, 4096, 128
    a.scale, a.num_splits, a.out, a.lse = 128 ** -0.5, 1, 0x4000, 0x5000
    for k_, v_ in kw.items():
        setattr(a, k_, v_)
    return a


@pytest.mark.parametrize("kw,ckw,stats,code,msg", [
    (dict(D=96), {}, 0, -2, "unsupported head dim / group size"),
    (dict(Hq=136), {}, 0, -2, "unsupported head dim / group size"),
    (dict(Hq=30), {}, 0, -1, "Hq must be a multiple of Hkv"),
    (dict(T=0), {}, 0, -1, "sizes must be positive"),
    (dict(T=2 ** 31 - 127), {}, 0, -2, "T up to 2^31 - 128"),
    (dict(k_st=136), {}, 0, -1, "k strides must be multiples of 16"),
    (dict(v=0x3008), {}, 0, -1, "v must be 16-byte aligned"),
    (dict(k=0), {}, 0, -1, "k must be 16-byte aligned"),
    (dict(k_st=1 << 24), {}, 0, -2, "k: token stride"),
    (dict(v_st=-128), {}, 0, -2, "v: token stride"),
    ({}, dict(format=2), 0, -1, "format e4m3 or int8"),
    ({}, dict(k_scale=0), 0, -1, "k_scale and v_scale"),
    (dict(out=0), {}, 0, -1, "out is required"),
    (dict(out=0x4008), {}, 0, -1, "must be 16-byte aligned"),
    (dict(out_f32=0x4008), {}, 0, -1, "must be 16-byte aligned"),
    (dict(num_splits=4, part_acc=0x4004, part_ml=0x4000), {}, 0, -1, "must be 16-byte aligned"),
    (dict(num_splits=4, part_acc=0x4000, part_ml=0x4008), {}, 0, -1, "must be 16-byte aligned"),
    ({}, {}, 1, -1, "stats needs blk_max"),
    (dict(num_splits=4), {}, 0, -1, "split partial buffers"),
    (dict(num_splits=257), {}, 0, -1, "num_splits <= 256"),
    (dict(p_out=0x100), {}, 0, -2, "no fp16 P"),
    (dict(block_idx=0x100), {}, 0, -1, "block_cnt is required"),
    (dict(seq_lens=0x100), {}, 0, -1, "seq_lens needs num_splits >= 2"),
    (dict(seq_lens=0x100, num_splits=2, part_acc=0x10, part_ml=0x10, B=257), {}, 0, -2, "seq_lens: B <= 256"),
    (dict(seq_lens=0x100, num_splits=2, part_acc=0x10, part_ml=0x10), {}, 0, -1, "seq_lens needs counts"),
    (dict(seq_lens=0x100, num_splits=2, part_acc=0x10, part_ml=0x10, T=(1 << 27) + 1), dict(counts=0x10), 0, -2, "T up to 2^27"),
    (dict(seq_lens=0x100, num_splits=2, part_acc=0x10, part_ml=0x10, block_idx=0x100, block_cnt=0x100,
          max_blocks=(1 << 21) + 1), dict(counts=0x10), 0, -2, "max_blocks up to 2^21"),
    (dict(list_partition=1), {}, 0, -1, "list_partition 1 partitions"),
    (dict(block_table=0x100, num_pages=4, bt_stride=63), {}, 0, -1, "paged cache"),
])
def test_decode8_refusals(kw, ckw, stats, code, msg):
    c = Cache8Args()
    c.k_scale, c.v_scale = 0x100, 0x200
    for k_, v_ in ckw.items():
        setattr(c, k_, v_)
    lib = _native.lib()
    assert lib.kvskip_decode8(ctypes.byref(_attn(**kw)), ctypes.byref(c), stats, None) == code
    assert msg in lib.kvskip_last_error().decode()


def test_decode8_null():
    lib = _native.lib()
    assert lib.kvskip_decode8(None, None, 0, None) == -1
    assert lib.kvskip_decode8(ctypes.byref(_attn()), None, 0, None) == -1


def _page(**kw):
    p = PageArgs()
    for f in ("seq_lens", "new_lens", "held", "block_table", "free_pages", "free_count", "slots", "starts", "held_out",
              "free_count_out", "short_out"):
        setattr(p, f, 0x1000)
    p.B, p.width, p.bt_stride, p.num_pages, p.rows = 4, 10, 10, 100, 64
    for k_, v_ in kw.items():
        setattr(p, k_, v_)
    return p


@pytest.mark.parametrize("kw,code,msg", [
    (dict(B=0), -1, "sizes must be positive"), (dict(width=0), -1, "sizes must be positive"),
    (dict(num_pages=0), -1, "sizes must be positive"), (dict(rows=-1), -1, "sizes must be positive"),
    (dict(B=2049), -2, "B <= 2048"), (dict(B=2048, rows=1 << 20), -2, "below 2^31"),
    (dict(num_pages=1 << 25), -2, "below 2^31"), (dict(B=2048, width=1 << 20, bt_stride=1 << 20), -2, "below 2^31"),
    (dict(bt_stride=9), -1, "must not overlap"), (dict(starts=0), -1, "null tensor"), (dict(slots=0), -1, "null tensor"),
    (dict(rows=1 << 20), -1, "work of kvskip_page_work_ints"),
])
def test_page_map_refusals(kw, code, msg):
    lib = _native.lib()
    assert lib.kvskip_page_map(ctypes.byref(_page(**kw)), None) == code
    assert msg in lib.kvskip_last_error().decode()
    assert lib.kvskip_page_map(None, None) == -1


def test_page_work():
    lib = _native.lib()
    assert lib.kvskip_page_work_ints(4, 64) == 0 and lib.kvskip_page_work_ints(4, 1 << 20) > 0
    assert lib.kvskip_page_work_ints(0, 1) == -1 and lib.kvskip_page_work_ints(5000, 1) == -1


def _write(**kw):
    p = WriteArgs()
    for f in ("k", "v", "slot_map", "k_pool", "v_pool", "k_scale", "v_scale"):
        setattr(p, f, 0x1000)
    p.N, p.Hkv, p.D, p.num_pages, p.format = 5, 8, 128, 100, 0
    p.k_sn = p.v_sn = 1024
    p.k_sh = p.v_sh = 128
    p.kp_sb = p.vp_sb = 8 * 64 * 128
    p.kp_sh = p.vp_sh = 64 * 128
    p.kp_st = p.vp_st = 128
    for k_, v_ in kw.items():
        setattr(p, k_, v_)
    return p


@pytest.mark.parametrize("kw,code,msg", [
    (dict(N=-1), -1, "sizes must be positive"), (dict(Hkv=0), -1, "sizes must be positive"),
    (dict(D=80), -2, "D in {64, 128}"), (dict(num_pages=1 << 25), -2, "below 2^31"), (dict(format=3), -1, "format"),
    (dict(slot_map=0), -1, "null tensor"), (dict(k_scale=0), -1, "k_scale and v_scale"),
    (dict(k=0x1008), -1, "k, v rows must be 16-byte aligned"), (dict(v_sh=100), -1, "k, v rows must be 16-byte aligned"),
    (dict(kp_st=136), -1, "pool rows must be 16-byte aligned"), (dict(v_pool=0x1004), -1, "pool rows must be 16-byte"),
    (dict(N=(1 << 21) + 1), -2, "N up to 2^21"), (dict(N=1 << 20, Hkv=257), -2, "N * Hkv up to 2^28"),
    (dict(Hkv=1 << 23), -2, "N * Hkv up to 2^28"), (dict(k_sn=1 << 24), -2, "row strides"), (dict(vp_st=-16), -2, "row strides"),
])
def test_cache_write_refusals(kw, code, msg):
    lib = _native.lib()
    assert lib.kvskip_cache_write(ctypes.byref(_write(**kw)), None) == code
    assert msg in lib.kvskip_last_error().decode()
    assert lib.kvskip_cache_write(ctypes.byref(_write(N=0)), None) == 0


def test_python_refusals():
    q = torch.zeros(1, 8, 64, dtype=torch.bfloat16)
    k8 = torch.zeros(1, 8, 64, 64, dtype=torch.int8)
    s = torch.ones(1, 8, 1)
    with pytest.raises(RuntimeError, match="belong together"):
        K.decode(q, k8, k8, 1.0, k_scale=s, num_splits=1)
    with pytest.raises(RuntimeError, match="read with V"):
        K.decode(q, k8, k8, 1.0, k_scale=s, v_scale=s, stats=True, load_v=False, num_splits=1)
    with pytest.raises(RuntimeError, match=r"q must be CUDA bf16"):
        ext.decode8(q, k8, k8, s, s, 1.0)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="seq_lens: contiguous CUDA int32"):
        ext.page_map(i, i, i, i.view(1, 1), i, i, i)
    with pytest.raises(RuntimeError, match="must be CUDA bf16"):
        ext.cache_write(q, q, i, k8, k8, s, s)
    with pytest.raises(RuntimeError, match="must be a tensor"):
        ext.cache_write(None, q, i, k8, k8)


def test_oracle_scale():
    for fmt, qmax in OPG.QMAX.items():
        for amax in (1e-45, 1e-38, 0.3, qmax, qmax * 1.01, qmax * 2 ** -9, 3e38):
            s = OPG.pow2_scale(amax, fmt)
            assert math.log2(s) == int(math.log2(s)) and amax <= qmax * s
            assert s == 2.0 ** -126 or amax > qmax * s / 2
        assert OPG.pow2_scale(0.0, fmt) == 0.0


def test_oracle_codes():
    """Every finite code comes back; halves go to even; torch's own conversion agrees."""
    c = torch.arange(256, dtype=torch.uint8)
    f = c[(c & 127) != 127]
    assert torch.equal(OPG.encode(OPG.decode_values(f, "e4m3"), "e4m3"), f)
    assert torch.equal(OPG.encode(OPG.decode_values(c, "int8").clamp(min=-127), "int8"), c.view(torch.int8).clamp(min=-127).view(torch.uint8))
    x = torch.linspace(-448, 448, 20011, dtype=torch.float64)
    assert torch.equal(OPG.encode(x.float().double(), "e4m3"), x.float().to(torch.float8_e4m3fn).view(torch.uint8))
    assert OPG.encode(torch.tensor([0.5, 1.5, 2.5], dtype=torch.float64), "int8").tolist() == [0, 2, 2]


def test_oracle_step():
    slots, starts, short, table, free, held, count = OPG.page_map(
        [65, 0, 3], [2, 0, 3], [1, 2, 0], [[4, 9], [6, 7], [9, 9]], [1, 0, 0, 0, 0, 0, 0, 0], 1, 6)
    # request 1 gives 6 and 7 back on [1]; request 0 takes 7, request 2 takes 6
    assert table == [[4, 7], [6, 7], [6, 9]] and held == [2, 0, 1] and count == 1 and short == 0
    assert slots == [4 * 64 + 63, 7 * 64, 6 * 64, 6 * 64 + 1, 6 * 64 + 2, -1] and starts == [0, 2, 2, 5]

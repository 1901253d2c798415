"""CPU: what attention over a step's rows and rotations refuse, before any launch; the sizes of a plan; the oracle on a case by hand."""

import ctypes

import pytest
import torch

from kvskip_amd import _native, ext, kvskip as K
from kvskip_amd._native import AttendArgs, AttendPlanArgs, RopeArgs
from kvskip_amd.paged import PagedCache
from oracle import attend as OA


def plan(**kw):
    p = AttendPlanArgs()
    p.starts = p.seq_lens = p.work = p.positions = 0x1000
    p.B, p.rows, p.Hq, p.Hkv, p.T = 3, 100, 32, 8, 4096
    for x, y in kw.items():
        setattr(p, x, y)
    return p


def test_struct_sizes():
    lib = _native.lib()
    for i, s in ((8, AttendPlanArgs), (9, AttendArgs), (10, RopeArgs)):
        assert lib.kvskip_struct_size(i) == ctypes.sizeof(s)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(B=0), -1, "sizes must be positive"), (dict(rows=0), -1, "sizes must be positive"),
    (dict(Hq=30), -1, "Hq must be a multiple of Hkv"), (dict(B=2049), -2, "B <= 2048"),
    (dict(shared=65), -2, "at most 64 shared prefixes"), (dict(shared=-1), -2, "at most 64"),
    (dict(shared=1, shared_T=0), -1, "shared_T >= 1"), (dict(shared=1, shared_T=64), -1, "null tensor"),
    (dict(T=(1 << 27) + 1), -2, "T and shared_T up to 2^27"), (dict(rows=(1 << 21) + 1), -2, "rows to 2^21"),
    (dict(rows=1 << 20, Hq=128), -2, "rows * Hq to 2^26"), (dict(max_rows=-1), -1, "max_rows >= 0"),
    (dict(window=-1), -1, "window >= 0"), (dict(work=0), -1, "work must be 16-byte aligned"),
    (dict(work=0x1004), -1, "work must be 16-byte aligned"), (dict(positions=0), -1, "null tensor"),
    (dict(starts=0), -1, "null tensor")])
def test_plan_validation(kw, code, msg):
    lib = _native.lib()
    assert lib.kvskip_attend_plan(ctypes.byref(plan(**kw)), None) == code
    assert msg in lib.kvskip_last_error().decode()


def attend_args(p=None, **kw):
    a = AttendArgs()
    a.plan = p or plan()
    for f in ("q", "k", "v", "k_scale", "v_scale", "block_table", "out", "lse", "part_acc", "part_ml"):
        setattr(a, f, 0x1000)
    a.q_sn, a.q_sh = 32 * 128, 128
    a.k_sb, a.k_sh, a.k_st = 8 * 64 * 128, 64 * 128, 128
    a.v_sb, a.v_sh, a.v_st = a.k_sb, a.k_sh, a.k_st
    a.bt_stride, a.scale, a.D, a.num_pages, a.format = 64, 0.1, 128, 10, 0
    for x, y in kw.items():
        setattr(a, x, y)
    return a


@pytest.mark.parametrize("kw,code,msg", [
    (dict(D=96), -2, "D in {64, 128}"), (dict(format=2), -1, "format e4m3 or int8"), (dict(q=0), -1, "q rows must be 16-byte"),
    (dict(q_sh=4), -1, "q rows must be 16-byte"), (dict(k=0x1008), -1, "k must be 16-byte aligned"),
    (dict(v_st=8), -1, "v strides must be multiples of 16"), (dict(k_st=1 << 24), -2, "token stride"),
    (dict(k_scale=0), -1, "k_scale and v_scale"), (dict(num_pages=0), -1, "num_pages >= 1"),
    (dict(bt_stride=63), -1, "block_table rows of ceil(T / 64) pages"), (dict(out=0), -1, "null tensor"),
    (dict(part_acc=0x1008), -1, "16-byte aligned"), (dict(softcap=-1.0), -1, "softcap"),
    (dict(softcap=float("nan")), -1, "softcap"), (dict(softcap=float("inf")), -1, "softcap"),
    (dict(p=plan(shared=2, shared_T=64)), -1, "shared_table rows"), (dict(p=plan(work=0x1001)), -1, "work must be")])
def test_attend_validation(kw, code, msg):
    lib = _native.lib()
    assert lib.kvskip_attend(ctypes.byref(attend_args(**kw)), None) == code
    assert msg in lib.kvskip_last_error().decode()


def rope_args(**kw):
    a = RopeArgs()
    a.q = a.k = a.q_out = a.k_out = a.positions = a.inv_freq = 0x1000
    a.rows, a.Hq, a.Hkv, a.D, a.rot, a.axes = 10, 8, 2, 128, 128, 1
    a.sections[0] = 64
    a.eps = 1e-6
    for x, y in kw.items():
        if x == "sections":
            for i, n in enumerate(y):
                a.sections[i] = n
        else:
            setattr(a, x, y)
    return a


@pytest.mark.parametrize("kw,code,msg", [
    (dict(D=12), -2, "D a multiple of 8"), (dict(D=264), -2, "D a multiple of 8"), (dict(rot=12), -2, "rotated elements"),
    (dict(rot=136), -2, "rotated elements"), (dict(axes=5), -1, "1 to 4 axes"), (dict(sections=[63]), -1, "sections of rot / 2"),
    (dict(axes=2, sections=[65, -1]), -1, "sections of rot / 2"), (dict(eps=-1.0), -1, "eps >= 0"), (dict(Hq=0), -1, "positive"),
    (dict(q=0), -1, "null tensor"), (dict(positions=0), -1, "null tensor"), (dict(k_out=0), -1, "null tensor"),
    (dict(q=0x1004), -1, "rows of whole 8 bytes"), (dict(k_sn=2), -1, "rows of whole 8 bytes")])
def test_rope_validation(kw, code, msg):
    lib = _native.lib()
    assert lib.kvskip_norm_rope(ctypes.byref(rope_args(**kw)), None) == code
    assert msg in lib.kvskip_last_error().decode()


def test_nothing_to_rotate_launches_nothing():
    assert _native.lib().kvskip_norm_rope(ctypes.byref(rope_args(rows=0)), None) == 0


@pytest.mark.parametrize("rows,B,Hq,Hkv,shared,most", [(1, 1, 4, 4, 0, 1), (24, 24, 32, 8, 0, 1), (20000, 7, 28, 4, 3, 0),
                                                       (2 ** 21, 2048, 32, 8, 64, 0), (65536, 1, 1024, 1, 0, 1)])
def test_plan_sizes(rows, B, Hq, Hkv, shared, most):
    lib = _native.lib()
    p = plan(rows=rows, B=B, Hq=Hq, Hkv=Hkv, shared=shared, shared_T=64 * bool(shared), max_rows=most)
    work, part = lib.kvskip_attend_work_ints(ctypes.byref(p)), lib.kvskip_attend_part_rows(ctypes.byref(p))
    tiles = rows * (Hq // Hkv) // 128 + B
    assert work > 16 * tiles and work < 2 ** 31 and 0 < part < 2 ** 31
    p.Hq = 7
    assert lib.kvskip_attend_work_ints(ctypes.byref(p)) == (-1 if 7 % Hkv else lib.kvskip_attend_work_ints(ctypes.byref(p)))


def test_python_refusals():
    bt = torch.zeros(2, 4, dtype=torch.int32)
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="block_table, shared_table: int32"):
        K.attend_plan(i, i[:2], 4, bt, 8, 2)
    with pytest.raises(RuntimeError, match="block_table must be a tensor"):
        K.attend_plan(i, i[:2], 4, None, 8, 2)
    q = torch.zeros(4, 8, 64, dtype=torch.bfloat16)
    p = ext.AttendPlan(i, i, bt, None, 4, 8, 2, 0, 0)
    with pytest.raises(RuntimeError, match="q must be CUDA bf16"):
        K.attend(q, q, q, 1.0, p, q, q)
    with pytest.raises(RuntimeError, match="norm_rope: q must be CUDA bf16"):
        ext.norm_rope(q, q, i, q)


def test_paged_cache_prefix_refusals():
    c = PagedCache(1, 2, 1, 64, 3, 100, 8, device="cpu", shared=(100, 64))
    assert c.pools[0][0].shape[0] == 2 + 2 + 1 and c.shared_table.tolist() == [[2, 3], [4, -1]]
    assert c.free_pages.tolist() == [0, 1] and c.shared_of.tolist() == [-1] * 3
    for call in (lambda: c.plan_prefix(2, 5, 4), lambda: c.plan_prefix(0, 101, 4), lambda: c.plan_prefix(0, 0, 4),
                 lambda: c.write_prefix(0, 1, torch.zeros(65, 1, 64), None), lambda: c.write_prefix(0, -1, torch.zeros(5, 1, 64), None)):
        with pytest.raises(ValueError, match="prefix in 0..1"):
            call()
    assert c.shared_lens.tolist() == [0, 0]
    with pytest.raises(ValueError, match="capacity of each prefix"):
        PagedCache(1, 2, 1, 64, 3, 100, 8, device="cpu", shared=(0,))


def test_oracle_by_hand():
    """Two keys, one of them seen by the first row."""
    k = torch.zeros(1, 1, 64, 64, dtype=torch.int8)
    v = torch.zeros(1, 1, 64, 64, dtype=torch.int8)
    k[0, 0, 1, 0], v[0, 0, 0, 0], v[0, 0, 1, 0] = 2, 10, 30
    one = torch.ones(1, 1)
    q = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    q[:, 0, 0] = 1
    out, lse, mass, _, _ = OA.attend(q, k, v, one, one, 0.5, [0, 2], [2], torch.zeros(1, 1, dtype=torch.int32))
    e = torch.e
    assert out[0, 0, 0] == 10 and lse[0, 0] == 0
    assert abs(out[1, 0, 0] - (10 + 30 * e) / (1 + e)) < 1e-12 and abs(lse[1, 0] - torch.log(torch.tensor(1 + e).double())) < 1e-7
    assert OA.positions([0, 2, 3], [5, 1], 4) == [3, 4, 0, -1]
    r = OA.norm_rope(torch.tensor([[[3.0, 0, 0, 4.0]]]), torch.tensor([[1]]), torch.tensor([torch.pi / 2, 0.0]))
    assert torch.allclose(r, torch.tensor([[[0.0, 0, 3.0, 4.0]]]).double(), atol=1e-6)

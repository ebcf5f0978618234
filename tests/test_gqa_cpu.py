"""CPU: what grouped-query caches refuse, and their tables without a device."""
import ctypes as C
import re
from pathlib import Path

import numpy as np
import pytest

import cautreo_b200 as ct

BF16, INT8, E4M3 = ct.CT_KV_BF16, ct.CT_KV_INT8, ct.CT_KV_E4M3


@pytest.mark.parametrize("layout,rc", [
    ((0, 64, 16, BF16, 4, 2), ct.CT_ERR_ARG), ((257, 64, 16, BF16, 4, 2), ct.CT_ERR_ARG),
    ((1, 64, 24, BF16, 4, 2), ct.CT_ERR_ARG), ((1, 64, 16, BF16, 0, 2), ct.CT_ERR_ARG),
    ((1, 64, 1 << 20, BF16, 1 << 12, 2), ct.CT_ERR_ARG), ((1, 64, 16, BF16, 4, 1 << 28), ct.CT_ERR_ARG),
    ((1, 80, 16, BF16, 4, 2), ct.CT_ERR_UNSUPPORTED), ((1, 0, 16, BF16, 4, 2), ct.CT_ERR_UNSUPPORTED),
    ((1, 512, 16, BF16, 4, 2), ct.CT_ERR_UNSUPPORTED), ((1, 64, 16, ct.CT_KV_F32, 4, 2), ct.CT_ERR_UNSUPPORTED),
    ((1, 64, 16, ct.CT_KV_Q8_0, 4, 2), ct.CT_ERR_UNSUPPORTED)])
def test_layouts_refused(layout, rc):
    L = ct.lib()
    lay = ct.GqaLayout(*layout)
    a = 4096                                          # an address that is never read: the layout is refused first
    assert L.ct_kv_gqa_write_slots(C.byref(lay), a, a, a, a, 0, 0, BF16, a, 1, None) == rc
    assert L.ct_kv_gqa_read_slots(C.byref(lay), a, a, a, 1, a, a, 0, 0, BF16, None) == rc
    assert L.ct_kv_gqa_page_bounds(C.byref(lay), a, a, a, a, 1, a, a, None) == rc
    assert not L.ct_gqa_plan_create(C.byref(ct.GqaShape(lay, 1, 0, 0, 0.0)), 1, 0)
    assert L.ct_hal_cuda_last_error()


def test_arguments_refused():
    L = ct.lib()
    lay = ct.GqaLayout(2, 64, 16, INT8, 4, 2)
    a = 4096

    def write(pool=a, sc=a, k=a, v=a, ks=0, vs=0, src=BF16, slots=a, n=1):
        return L.ct_kv_gqa_write_slots(C.byref(lay), pool, sc, k, v, ks, vs, src, slots, n, None)

    for bad in (dict(pool=None), dict(pool=a + 8), dict(sc=None), dict(sc=a + 4), dict(k=None), dict(v=a + 2), dict(ks=64),
                dict(vs=132), dict(src=INT8), dict(slots=None)):
        assert write(**bad) == ct.CT_ERR_ARG, bad
    assert write(src=ct.CT_KV_F32, ks=130) == ct.CT_ERR_ARG
    assert write(n=0) == ct.CT_OK
    assert L.ct_kv_gqa_write_slots(None, a, a, a, a, 0, 0, BF16, a, 1, None) == ct.CT_ERR_ARG

    def read(slots=a, k=a, v=a, ks=0, dt=BF16):
        return L.ct_kv_gqa_read_slots(C.byref(lay), a, a, slots, 1, k, v, ks, 0, dt, None)

    for bad in (dict(slots=None), dict(k=None), dict(v=a + 8), dict(ks=100), dict(dt=E4M3)):
        assert read(**bad) == ct.CT_ERR_ARG, bad
    for i in range(4):
        args = [a, a, 1, a, a]
        args[i if i < 2 else i + 1] = None
        assert L.ct_kv_gqa_page_bounds(C.byref(lay), a, a, args[0], args[1], args[2], args[3], args[4], None) == ct.CT_ERR_ARG


@pytest.mark.parametrize("shape", [dict(hq=0), dict(hq=3), dict(order=2), dict(pages=0), dict(n_seq=1 << 31), dict(hq=1 << 17)])
def test_plans_refused(shape):
    lay = ct.GqaLayout(2, 64, 16, BF16, 4, shape.get("pages", 1 << 20))
    s = ct.GqaShape(lay, shape.get("hq", 4), 0, shape.get("order", 0), 0.0)
    assert not ct.lib().ct_gqa_plan_create(C.byref(s), shape.get("n_seq", 1), 0)
    assert ct.lib().ct_hal_cuda_last_error()


def test_handles_refused():
    L = ct.lib()
    cfg = ct.PagedConfig(2, 4, 8, 16, 0, 0, BF16, -1)
    assert not L.ct_kv_paged_create_gqa(None, 2, 64, 0)
    assert not L.ct_kv_paged_create_gqa(C.byref(cfg), 2, 80, 0)
    assert not L.ct_kv_paged_create_gqa(C.byref(ct.PagedConfig(2, 4, 8, 16, 100, 0, BF16, -1)), 2, 64, 0)
    assert not L.ct_kv_paged_create_gqa(C.byref(ct.PagedConfig(2, 4, 8, 16, 0, 0, ct.CT_KV_F32, -1)), 2, 64, 0)
    other = ct.PagedKV(2, 4, 8, 16, 64, device=-1)
    ids, n = np.array([0], np.uint32), np.array([1], np.uint32)
    a = 4096
    assert L.ct_kv_paged_append_kv(other.h, ids.ctypes.data, n.ctypes.data, 1, a, a, 0, 0, BF16) == ct.CT_ERR_UNSUPPORTED
    assert L.ct_kv_paged_gather_kv(other.h, ids.ctypes.data, ids.ctypes.data, n.ctypes.data, 1, a, a, BF16) == ct.CT_ERR_UNSUPPORTED
    assert L.ct_kv_paged_gqa_layout(other.h, C.byref(ct.GqaLayout())) == ct.CT_ERR_UNSUPPORTED
    kv = ct.GqaKV(2, 4, 8, 2, 64, 16, device=-1)
    assert L.ct_kv_paged_append_kv(kv.h, ids.ctypes.data, n.ctypes.data, 1, a, None, 0, 0, BF16) == ct.CT_ERR_ARG
    assert L.ct_kv_paged_append_kv(kv.h, ids.ctypes.data, n.ctypes.data, 1, a, a + 8, 0, 0, BF16) == ct.CT_ERR_ARG
    assert L.ct_kv_paged_append_kv(kv.h, ids.ctypes.data, n.ctypes.data, 1, a, a, 8, 0, BF16) == ct.CT_ERR_ARG
    assert L.ct_kv_paged_append_kv(kv.h, ids.ctypes.data, n.ctypes.data, 1, a, a, 0, 0, INT8) == ct.CT_ERR_ARG
    assert L.ct_kv_paged_append_kv(kv.h, ids.ctypes.data, n.ctypes.data, 1, a, a, 0, 0, BF16) == ct.CT_ERR_UNSUPPORTED   # tables only
    assert L.ct_kv_paged_append_projected(kv.h, ids.ctypes.data, n.ctypes.data, 1, a, a, 64, None, 0.0, 0) == ct.CT_ERR_UNSUPPORTED
    assert kv.seq_lens().tolist() == [0, 0]


def test_tables_without_a_device(tmp_path):
    kv = ct.GqaKV(3, 4, 8, 2, 64, 16, dtype=INT8, keep_bounds=True, device=-1)
    kv.append([0, 1], [33, 5])
    kv.fork(0, 2, 20)
    assert kv.seq_lens().tolist() == [33, 5, 20] and kv.bounds is None
    kv.save(tmp_path / "t.bin")
    back = ct.GqaKV.load(tmp_path / "t.bin", device=-1)
    assert np.array_equal(back.block_table(), kv.block_table())
    lay = back.layout
    assert (lay.n_kv_heads, lay.head_dim, lay.page_tokens, lay.kv_dtype) == (2, 64, 16, INT8)
    back.append([1], [1])
    assert back.seq_lens().tolist() == [33, 6, 20]
    plain = ct.PagedKV(2, 4, 8, 16, 64, device=-1)
    plain.save(tmp_path / "p.bin")
    with pytest.raises(RuntimeError):
        ct.GqaKV.load(tmp_path / "p.bin", device=-1)


def test_plans_of_too_many_steps_refused():
    """More steps in all than a worker's 32-bit share of them holds, although each sequence's and each head's are few enough."""
    for n_seq, hq in ((1 << 18, 256), (3000, 65280)):
        s = ct.GqaShape(ct.GqaLayout(256, 64, 16, BF16, 4, 1 << 13), hq, 0, 0, 0.0)
        if hq > 256:
            s.kv.max_pages_per_seq = 60000
        assert not ct.lib().ct_gqa_plan_create(C.byref(s), n_seq, 0)
        assert b"too many" in ct.lib().ct_hal_cuda_last_error()


def test_kernels_launched_early_load_coherently():
    """These kernels are resident while the one before them still writes what they read, so none of their loads may take the
    non-coherent path, nor be an intrinsic that is free to move above the wait."""
    csrc = Path(ct.__file__).resolve().parent / "csrc"
    sources = sorted(csrc.glob("gqa_*"))
    assert len(sources) >= 5
    for f in sources:
        assert not re.findall(r"__ldg\b|__ldc[agsv]\b|__ldlu\b|global\.nc\b|__restrict__", f.read_text()), f.name


def test_pages_of_every_size_may_move():
    """A cache takes pages of up to 512 tokens here (latent caches any number), so its compaction has to move them."""
    L, a = ct.lib(), 4096
    for tokens in (16, 256, 272, 512, 4096):
        assert L.ct_kv_paged_move_pages(a, a, a, a, a, 0, 16, tokens, None) == ct.CT_OK, tokens
        assert L.ct_kv_paged_move_pages(a, None, a, None, a, 0, 16, tokens, None) == ct.CT_OK, tokens
    assert L.ct_kv_paged_move_pages(a, None, a, a, a, 0, 16, 64, None) == ct.CT_ERR_ARG
    assert L.ct_kv_paged_move_pages(a, None, a, None, a, 0, 24, 64, None) == ct.CT_ERR_ARG

"""CPU: the host layer of the paged caches and the grouped-query plans over a device made of host memory, which can be made to
fail at any call (tests/fake_cuda.c)."""
import ctypes as C
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

import cautreo_b200 as ct
from cautreo_b200 import build as B

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    """The host sources linked with the fake device (-Bsymbolic: also where a CUDA runtime is loaded), the package's signatures
    declared on it."""
    so = tmp_path_factory.mktemp("fake") / "libfake.so"
    host = ROOT / "cautreo_b200" / "host"
    cc = shutil.which("gcc") or "gcc"
    r = subprocess.run([cc, *B.CC_FLAGS, "-Wno-sign-compare", "-shared", "-Wl,-Bsymbolic", "-o", str(so), str(ROOT / "tests" / "fake_cuda.c"),
                        *(str(host / f) for f in ("kv_paged.c", "gqa.c", "runtime.c")), "-lm", "-lpthread"],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    L = C.CDLL(str(so))
    for name, (res, args) in ct.SIGNATURES.items():
        if hasattr(L, name):
            f = getattr(L, name)
            f.restype, f.argtypes = res, args
    L.fake_fail.argtypes = [C.c_long]
    L.fake_pending.restype = L.fake_live.restype = L.fake_unfinished.restype = C.c_long
    return L


class Handle:
    """A handle of the fake device: 4 sequences of 8 pages of 16 tokens, bf16, 2 heads of 32 (or entries of 128 values)."""
    S, NP, P, H, D = 4, 20, 16, 2, 32
    W = H * D

    def __init__(self, L, gqa, bounds=True, n_pages=None, window=0, pages_per_seq=8):
        self.L, self.gqa, self.MP = L, gqa, pages_per_seq
        cfg = ct.PagedConfig(self.S, self.MP, n_pages or self.NP, self.P, 2 * self.W, window, ct.CT_KV_BF16, 0)
        self.h = (L.ct_kv_paged_create_gqa(C.byref(cfg), self.H, self.D, int(bounds)) if gqa else L.ct_kv_paged_create(C.byref(cfg)))
        self.np = n_pages or self.NP
        self.rng = np.random.default_rng(7)
        self.rows = [np.zeros((0, 2 * self.W), np.uint16) for _ in range(self.S)]

    def append(self, seqs, counts):
        x = self.rng.integers(0, 1 << 16, (sum(counts), 2 * self.W), dtype=np.uint16)
        s, c = np.array(seqs, np.uint32), np.array(counts, np.uint32)
        aligned = C.create_string_buffer(x.nbytes + 32)
        at = (C.addressof(aligned) + 31) // 16 * 16
        C.memmove(at, x.ctypes.data, x.nbytes)
        rc = self.L.ct_kv_paged_append(self.h, s.ctypes.data, c.ctypes.data, len(s), at, ct.CT_KV_BF16)
        if rc == 0:
            o = 0
            for q, n in zip(seqs, counts):
                self.rows[q] = np.concatenate((self.rows[q], x[o:o + n]))
                o += n
        return rc

    def fork(self, src, dst, n):
        rc = self.L.ct_kv_paged_fork(self.h, src, dst, n)
        if rc == 0:
            self.rows[dst] = self.rows[src][:n].copy()
        return rc

    def table(self):
        t = np.zeros((self.S, self.MP), np.int32)
        self.L.ct_kv_paged_block_table(self.h, t.ctypes.data)
        return t

    def check(self, mapped_only=False):
        """Host and device tables agree, every token (that is still mapped) reads back, references and free pages add up, bounds
        follow."""
        t = self.table()
        dev = np.ctypeslib.as_array(C.cast(self.L.ct_kv_paged_block_table_dev(self.h), C.POINTER(C.c_int32)), t.shape)
        assert np.array_equal(dev, t)
        lens = np.ctypeslib.as_array(C.cast(self.L.ct_kv_paged_seq_lens_dev(self.h), C.POINTER(C.c_int32)), (self.S,))
        assert lens.tolist() == [len(r) for r in self.rows]
        out = C.create_string_buffer(2 * 2 * self.W * self.P * self.MP + 32)
        at = (C.addressof(out) + 31) // 16 * 16
        for s, r in enumerate(self.rows):
            first = int(np.argmax(t[s] >= 0)) * self.P if mapped_only and (t[s] >= 0).any() else 0
            r = r[first:]
            if len(r) == 0 or (mapped_only and not (t[s] >= 0).any()):
                continue
            assert self.L.ct_kv_paged_gather(self.h, s, first, len(r), at, ct.CT_KV_BF16) == 0
            got = np.frombuffer((C.c_char * r.nbytes).from_address(at), np.uint16).reshape(r.shape)
            assert np.array_equal(got, r), s
        ids, n = np.unique(t[t >= 0], return_counts=True)
        assert [self.L.ct_kv_paged_page_refs(self.h, int(p)) for p in ids] == n.tolist()
        st = self.L.ct_kv_paged_stats(self.h)
        assert st.n_pages_live == len(ids) and st.n_pages_free == self.np - len(ids)
        if self.gqa and self.L.ct_kv_paged_bound_scales(self.h):
            bs = np.ctypeslib.as_array(C.cast(self.L.ct_kv_paged_bound_scales(self.h), C.POINTER(C.c_float)), (self.np, self.H))
            for s, r in enumerate(self.rows):
                for lp in range(-(-len(r) // self.P)):
                    if mapped_only and t[s, lp] < 0:
                        continue
                    assert (bs[t[s, lp]] == min(self.P, len(r) - lp * self.P)).all()

    def close(self):
        self.L.ct_kv_paged_destroy(self.h)


def test_an_error_is_reported_once(fake):
    """A call that failed (here a plan whose scratch does not fit) does not make the next call, which works, fail as well."""
    h = Handle(fake, True)
    assert h.append([0, 1], [20, 3]) == 0
    lay = ct.GqaLayout()
    assert fake.ct_kv_paged_gqa_layout(h.h, C.byref(lay)) == 0
    shape = ct.GqaShape(lay, 4, 0, 0, 0.0)
    for k in (1, 2, 3):                               # the scratch, its stream, its zeroes
        fake.fake_fail(k)
        assert not fake.ct_gqa_plan_create(C.byref(shape), 2, 0) and fake.fake_pending() < 0
        assert b"gqa scratch" in fake.ct_hal_cuda_last_error()
        assert h.append([0, 1], [1, 1]) == 0
        h.check()
    h.close()


@pytest.mark.parametrize("gqa", [False, True])
@pytest.mark.parametrize("again", [False, True])
def test_a_compaction_that_fails_changes_nothing(fake, gqa, again):
    """Each device call of a compaction fails once; afterwards the handle reads, appends and compacts as if it had not begun."""
    for k in range(1, 40):
        live = fake.fake_live()
        h = Handle(fake, gqa)
        order = np.random.default_rng(k).permutation(h.NP).astype(np.int32)
        assert fake.ct_kv_paged_set_free_order(h.h, order.ctypes.data) == 0
        assert h.append([0, 1, 2], [40, 17, 64]) == 0 and h.fork(2, 3, 37) == 0
        if again:                                     # buffers of an earlier compaction
            assert fake.ct_kv_paged_compact(h.h) == 0
            assert fake.ct_kv_paged_free_seq(h.h, 1) == 0
            h.rows[1] = h.rows[1][:0]
        h.check()
        held, before = fake.fake_live(), h.table()
        fake.fake_fail(k)
        rc = fake.ct_kv_paged_compact(h.h)
        failed = fake.fake_pending() < 0
        fake.fake_fail(-1)
        assert (rc != 0) == failed
        if failed:
            assert rc == ct.CT_ERR_CUDA and np.array_equal(h.table(), before) and fake.fake_live() <= held
            assert fake.ct_kv_paged_stats(h.h).n_compactions == again
        h.check()
        assert h.append([1, 3], [20, 30]) == 0
        h.check()
        assert fake.ct_kv_paged_compact(h.h) == 0
        h.check()
        t = h.table()
        assert sorted(set(t[t >= 0].tolist())) == list(range(len(set(t[t >= 0].tolist()))))
        h.close()
        assert fake.fake_live() == live
        if not failed:
            break
    assert not failed and k > 4


def test_page_lists_of_any_length_are_refused_or_end(fake):
    """Entries of a row are counted in 32 bits by 256 threads, so lists that long are refused, not written without an end."""
    lay = ct.GqaLayout(1, 32, 16, ct.CT_KV_BF16, 4, 4)
    shape = ct.GqaShape(lay, 1, 0, 0, 0.0)
    plan = fake.ct_gqa_plan_create(C.byref(shape), 1, 0)
    a = 4096                                          # never read: the fake device computes nothing
    for n, rc in ((1, 0), (1 << 20, 0), (0x7FFFFFFF, 0), (0x80000000, ct.CT_ERR_ARG), (0xFFFFFFFF, ct.CT_ERR_ARG)):
        runs = fake.fake_runs()
        assert fake.ct_attn_gqa_select_pages(plan, a, 0, a, a, a, a, n, 0, 0, a, None) == rc, n
        assert fake.ct_attn_gqa_decode_selected(plan, a, 0, a, None, a, a, a, n, a, None, None) == rc, n
        assert fake.fake_runs() == runs + (2 if rc == 0 else 0)
    fake.ct_gqa_plan_destroy(plan)


def test_a_shared_page_gets_its_bounds_once_when_loaded(fake, tmp_path):
    """A checkpoint of forked sequences: every mapped page once in the call that makes the bounds, however many sequences map it
    (one block a listed page and head: entries of all tables would pass what a launch takes)."""
    h = Handle(fake, True)
    assert h.append([0], [7 * h.P + 3]) == 0
    for s in (1, 2, 3):
        assert h.fork(0, s, 7 * h.P + s - 1) == 0
    assert fake.ct_kv_paged_save(h.h, str(tmp_path / "f.bin").encode()) == 0
    back = Handle(fake, True)
    back.close()
    back.h, back.rows = fake.ct_kv_paged_load(str(tmp_path / "f.bin").encode(), 0), h.rows
    back.check()
    assert fake.fake_listed() == len(set(back.table()[back.table() >= 0].tolist())) == 10 and fake.fake_listed_twice() == 0
    back.close()
    h.close()


@pytest.mark.parametrize("gqa", [False, True])
def test_a_new_handle_leaves_nothing_running(fake, gqa, tmp_path):
    """Creating and loading work on the default stream, which the stream that the handle is given next need not wait for: what
    they set (zeroes, tables, bounds) is there when they return."""
    h = Handle(fake, gqa)
    assert fake.fake_unfinished() == 0
    assert h.append([0, 1], [40, 17]) == 0 and fake.fake_unfinished() > 0
    assert fake.ct_kv_paged_save(h.h, str(tmp_path / "f.bin").encode()) == 0
    h.close()
    h.h = fake.ct_kv_paged_load(str(tmp_path / "f.bin").encode(), 0)
    assert fake.fake_unfinished() == 0
    h.check()
    h.close()


def state(h):
    """Everything of a handle that a call can change on the host."""
    L = h.L
    st = L.ct_kv_paged_stats(h.h)
    last = np.zeros(h.S, np.uint64)
    lens = np.zeros(h.S, np.uint32)
    L.ct_kv_paged_last_access(h.h, last.ctypes.data)
    L.ct_kv_paged_seq_lens(h.h, lens.ctypes.data)
    return (h.table().tolist(), lens.tolist(), last.tolist(), [getattr(st, n) for n, _ in st._fields_],
            [L.ct_kv_paged_page_refs(h.h, p) for p in range(h.np)], L.ct_kv_paged_evict_log(h.h, None, 0))


@pytest.mark.parametrize("gqa", [False, True])
@pytest.mark.parametrize("window", [0, 40])
def test_an_append_without_room_changes_nothing(fake, gqa, window):
    """The pool or a table row is full in the middle of the call, pages evicted and used again before that among them: the call
    is refused as a whole, and works when there is room."""
    h = Handle(fake, gqa, n_pages=11, window=window)
    assert h.append([0, 1, 2], [33, 20, 16]) == 0
    h.fork(0, 3, 20)
    for seqs, counts in (([0, 1], [100, 3]), ([3, 0], [1, 129]), ([2, 2], [60, 60]), ([1, 0, 3], [30, 126, 30])):
        before = state(h)
        assert h.append(seqs, counts) == ct.CT_ERR_FULL, (seqs, counts)
        assert state(h) == before
        h.check(mapped_only=True)
    assert fake.ct_kv_paged_free_seq(h.h, 2) == 0
    h.rows[2] = h.rows[2][:0]
    assert h.append([1, 2], [5, 17]) == 0
    h.check(mapped_only=True)
    h.close()


@pytest.mark.parametrize("gqa", [False, True])
def test_an_append_that_fails_on_the_device_changes_nothing(fake, gqa):
    """Each device call of an append fails once (the staging buffers grow in it).  Up to the launch that writes the tokens the
    handle stays as it was, on the host and on the device; the launch of the bounds comes after that, and the tokens are there."""
    last = 0
    for k in range(1, 40):
        h = Handle(fake, gqa, n_pages=300, pages_per_seq=200)
        assert h.append([0, 1], [40, 17]) == 0 and h.fork(0, 2, 21) == 0
        before = state(h)
        fake.fake_fail(k)
        rows = [r.copy() for r in h.rows]
        rc = h.append([0, 1, 3], [2000, 9, 2500])
        failed = fake.fake_pending() < 0
        fake.fake_fail(-1)
        assert (rc != 0) == failed
        if failed and state(h) != before:             # only the bounds are missing
            assert gqa and k == last + 1
            h.close()
            break
        if failed:
            last = k
            assert all(np.array_equal(a, b) for a, b in zip(h.rows, rows))
            h.check()
            assert h.append([0, 1, 3], [2000, 9, 2500]) == 0
        h.check()
        h.close()
        if not failed:
            break
    assert last >= 5

"""Attention over the cache without a GPU: sizes at the ends of what the rules divide by and choose between, and what is refused."""
import ctypes as C
import os
import subprocess
import sys

import pytest
import torch

from vectorlink_gpu import _native as nv
from vectorlink_gpu import attention

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vectorlink-gpu_amd")

# every call that says how much workspace a call takes, and the calls, of no rows: in a process of its own, which a division by zero ends
NO_ROWS = """
import ctypes as C
import sys
sys.path.insert(0, sys.argv[1])
from vectorlink_gpu import _native as nv
lib = nv.lib()
parts = dict(keys=256, key_scales=256, values=256, value_scales=256, bounds=256, bound_scales=256)
for dim in (32, 64, 96, 128, 192, 256):
    for (heads, group) in ((1, 1), (8, 4), (2, 20)):
        cache = C.byref(nv.Cache(pages=10, heads=heads, dim=dim, **parts))
        for blocks in (0, 1, 7, 8, 64, 40_000):
            for sequences in (0, 1, 5):
                tokens = C.byref(nv.Tokens(rows=0, sequences=sequences, blocks=blocks, table_stride=blocks, table=256, lengths=256, offsets=256))
                for type in (1, 2, 3):
                    for form in (0, 1, 2) if dim * type <= 256 else (0, 1):
                        q = C.byref(nv.Queries(heads=heads * group, row_stride=0, head_stride=0, scale=1.0, type=type, causal=1, form=form))
                        assert lib.vl_attend_form(cache, tokens, q) in ((1, 2) if form == 0 else (form,))
                        assert lib.vl_attend_workspace_bytes(cache, tokens, q) == 0
                        assert lib.vl_select_blocks_workspace_bytes(cache, tokens, q, 4) == 0
                        assert lib.vl_attend_blocks_workspace_bytes(cache, tokens, q, 4) == 0
                        assert lib.vl_attend_selected_workspace_bytes(cache, tokens, q, 4) == 0
                        assert lib.vl_attend(cache, tokens, q, None, 0, None) == 0
                        assert lib.vl_attend_selected(cache, tokens, q, 4, None, None, 0, None) == 0
print("all answered")
"""


def test_no_rows_in_every_form():
    r = subprocess.run([sys.executable, "-c", NO_ROWS, PKG], capture_output=True, text=True)
    assert r.returncode == 0 and "all answered" in r.stdout, (r.returncode, r.stderr[-500:])


def native(rows, sequences, blocks, heads=8, group=4, dim=128, type=1):
    parts = dict(keys=256, key_scales=256, values=256, value_scales=256, bounds=256, bound_scales=256)
    return (C.byref(nv.Cache(pages=10, heads=heads, dim=dim, **parts)),
            C.byref(nv.Tokens(rows=rows, sequences=sequences, blocks=blocks, table_stride=blocks, table=256, lengths=256, offsets=256)),
            C.byref(nv.Queries(heads=heads * group, row_stride=0, head_stride=0, scale=1.0, type=type, causal=1, form=0)))


def test_sequences_without_rows_count_for_nothing():
    """A batch with a place for each of many sequences, of which few have new tokens, is answered as those few are."""
    lib = nv.lib()
    for rows in (1, 3, 10, 63):
        for blocks in (16, 128, 2048):
            for kw in (dict(), dict(heads=1, group=1, dim=64), dict(type=2), dict(dim=256)):
                alone = native(rows, rows, blocks, **kw)
                want = (lib.vl_attend_form(*alone), lib.vl_attend_workspace_bytes(*alone))
                assert want[0] == 1
                for sequences in (rows + 1, 64, 256, 4096):
                    among = native(rows, sequences, blocks, **kw)
                    assert (lib.vl_attend_form(*among), lib.vl_attend_workspace_bytes(*among)) == want, (rows, sequences, blocks, kw)


def test_scales_beyond_float32_are_refused():
    lib = nv.lib()
    parts = dict(keys=256, key_scales=256, values=256, value_scales=256, bounds=256, bound_scales=256)
    cache = C.byref(nv.Cache(pages=10, heads=2, dim=128, **parts))
    tokens = C.byref(nv.Tokens(rows=3, sequences=3, blocks=4, table_stride=4, table=256, lengths=256))
    for scale in (1e39, -2.4e38, 1e300, float("inf"), float("nan")):
        q = C.byref(nv.Queries(heads=8, row_stride=1024, head_stride=128, queries=256, out=256, scale=scale, type=1, causal=1))
        assert lib.vl_attend(cache, tokens, q, 256, 1 << 40, None) == -1 and b"scale" in lib.vl_last_error()
        assert lib.vl_attend_blocks(cache, tokens, q, 256, 4, 256, 1 << 40, None) == -1
        assert lib.vl_attend_selected(cache, tokens, q, 4, 256, 256, 1 << 40, None) == -1


class Sizes:
    """Stands for a cache where only its sizes are looked at."""
    (pages, heads, dim) = (4, 2, 64)
    keys = torch.zeros(1)
    _ref = None


def test_what_asks_for_a_gradient_is_refused():
    """There is none: it would be lost without a word."""
    q = torch.zeros((3, 4, 64), requires_grad=True)
    (table, lengths) = (torch.zeros((3, 4), dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
    blocks = torch.zeros((3, 2, 1), dtype=torch.int32)
    calls = [lambda: attention.attend(q, Sizes, table, lengths), lambda: attention.select_blocks(q, Sizes, table, lengths, 2),
             lambda: attention.attend_blocks(q, Sizes, table, lengths, blocks), lambda: attention.attend_selected(q, Sizes, table, lengths, 2),
             lambda: attention.KVCache.write(Sizes, q[:, :2], q[:, 2:].detach(), table, lengths),
             lambda: attention.KVCache.write(Sizes, q[:, :2].detach(), q[:, 2:], table, lengths)]
    for call in calls:
        with pytest.raises(AssertionError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):  # as far as it goes without one
            call()


class On:
    """Stands for a tensor on a GPU of that number."""
    is_cuda = True

    def __init__(self, gpu):
        self.gpu = gpu

    def get_device(self):
        return self.gpu


def test_tensors_of_another_gpu_are_refused(monkeypatch):
    """Kernels run on the current GPU, on its stream: what lies on another would be read across GPUs, if it can be."""
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda gpu: 100 + gpu, raising=False)
    assert nv.require_one_gpu(On(1), None, On(1)) == 1 and nv.require_one_gpu(On(0)) == 0
    assert nv.stream_on(1, 1).value == 101
    for bad in ((On(1), On(0)), (On(0), None, On(1)), (On(1), torch.zeros(3)), (torch.zeros(3), On(1)), (torch.zeros(3),)):
        with pytest.raises(RuntimeError, match="GPU"):
            nv.require_one_gpu(*bad)
    for bad in ((0,), (1, 0), (0, 0)):
        with pytest.raises(RuntimeError, match="GPU"):
            nv.stream_on(*bad)


def test_every_call_asks_where_its_tensors_are(monkeypatch):
    """The cache, what is written or asked, tables, lengths, offsets and lists; and for the stream of that GPU."""
    (seen, gpus) = ([], [])

    class Library:
        def __getattr__(self, name):
            return lambda *args: 0

    class Cache(Sizes):
        gpu = 5

    monkeypatch.setattr(nv, "lib", Library)
    monkeypatch.setattr(nv, "require_one_gpu", lambda *tensors: seen.extend(id(t) for t in tensors) or 7)
    monkeypatch.setattr(nv, "stream_on", lambda *of: gpus.extend(of))
    (q, kv) = (torch.zeros((3, 4, 64)), torch.zeros((3, 2, 64)))
    (table, lengths, offsets) = (torch.zeros((3, 4), dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32))
    blocks = torch.zeros((3, 2, 1), dtype=torch.int32)
    calls = [(lambda: attention.attend(q, Cache, table, lengths, offsets), [q, table, lengths, offsets]),
             (lambda: attention.select_blocks(q, Cache, table, lengths, 2, offsets), [q, table, lengths, offsets]),
             (lambda: attention.attend_blocks(q, Cache, table, lengths, blocks, offsets), [q, table, lengths, offsets, blocks]),
             (lambda: attention.attend_selected(q, Cache, table, lengths, 2, offsets), [q, table, lengths, offsets]),
             (lambda: attention.KVCache.write(Cache, kv, kv, table, lengths, offsets), [kv, table, lengths, offsets]),
             (lambda: attention.KVCache.read(Cache, table, lengths, 3, offsets), [table, lengths, offsets]),
             (lambda: attention.KVCache.read_bounds(Cache, lengths), [lengths])]
    for call, tensors in calls:
        seen.clear()
        gpus.clear()
        call()
        assert {id(t) for t in tensors} <= set(seen) and set(gpus) == {7, 5}


def test_launches_of_a_choice_and_its_attention():
    """One launch or several, by what was measured: (tokens, heads, dim, type, blocks, count) on either side.  One launch has no workspace."""
    lib = nv.lib()

    def one(rows, heads, dim, type, blocks, count):
        (cache, tokens, q) = native(rows, rows, blocks, heads=heads, dim=dim, type=type)
        return lib.vl_attend_selected_workspace_bytes(cache, tokens, q, count) == 0

    for sizes in ((1, 8, 128, 1, 256, 16), (1, 8, 128, 1, 1024, 32), (1, 8, 128, 1, 1024, 64), (1, 4, 256, 1, 1024, 16), (8, 8, 128, 1, 1000, 64),
                  (8, 8, 128, 2, 1000, 16), (1, 8, 128, 3, 1000, 16), (32, 8, 128, 1, 512, 32), (32, 8, 128, 1, 8000, 256), (16, 8, 128, 1, 1000, 256)):
        assert one(*sizes), sizes
    for sizes in ((1, 8, 128, 1, 2048, 32), (1, 8, 128, 1, 1040, 16), (1, 4, 64, 1, 2048, 32), (1, 8, 128, 1, 256, 64), (8, 8, 128, 1, 300, 256),
                  (8, 8, 64, 1, 300, 256), (8, 8, 256, 1, 1000, 256), (1, 8, 128, 3, 256, 32), (4, 8, 128, 2, 300, 64), (16, 8, 128, 1, 300, 256)):
        assert not one(*sizes), sizes

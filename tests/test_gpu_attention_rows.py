"""Rows before the first offset and behind the last belong to no sequence: no call writes what would be theirs, whatever the
buffers, lists and workspaces hold there.  Calls through the C ABI, as only it takes the caller's own buffers."""
import pytest
import torch

import attention_reference as ref
from test_gpu_attention import DEV, ends, filled, queries_for
from test_gpu_attention_many import check, dense
from vectorlink_gpu import _native as nv
from vectorlink_gpu import attention

pytestmark = pytest.mark.gpu
MARK = -3.0
MARKED = 123_456


class Call:
    """One call's buffers, marked: 40 rows or so on two sequences, of which some in front and some behind belong to none."""

    def __init__(self, counts, rows, heads=2, group=3, dim=64, lengths=(3000, 300), blocks=None, before=0, dtype=torch.bfloat16):
        (self.cache, self.table, self.lengths, gen) = filled(list(lengths), heads, dim, 5, dtype, blocks=blocks)
        self.at = ends(counts) + before
        self.mine = slice(before, before + sum(counts))
        self.q = queries_for(rows, heads * group, dim, gen, dtype)
        (self.out, self.lse) = (torch.full_like(self.q, MARK), torch.full(self.q.shape[:2], MARK, device=DEV))
        self.tokens = attention._tokens(rows, self.table, self.lengths, self.at)

    def native(self, form=None):
        return attention._queries(self.q, self.cache, None, True, self.out, self.lse, form)

    def list(self, count):
        return torch.full((self.q.size(0), self.cache.heads, count), MARKED, dtype=torch.int32, device=DEV)

    @staticmethod
    def workspace(need):
        """Full of numbers, as recycled memory is."""
        return torch.full((max(4, nv.check(need)) // 4,), 5.0, device=DEV)

    def others(self, t):
        return torch.cat((t[:self.mine.start], t[self.mine.stop:]))

    def check(self, blocks=None, lse=True):
        assert (self.others(self.out) == MARK).all() and (self.others(self.lse) == MARK).all()
        want = ref.attention(self.q, self.cache, self.table, self.lengths, self.at, blocks=None if blocks is None else blocks.cpu())
        ref.check_attention(self.out[self.mine], tuple(t[self.mine] for t in want), self.q.dtype)
        if lse:
            assert ((self.lse[self.mine].cpu().double() - want[1][self.mine]).abs() <= (want[2][self.mine] + 16) * 2.0 ** -24).all()


CASES = [dict(counts=[7, 5], rows=40), dict(counts=[7, 5], rows=12 + 9, before=9), dict(counts=[1, 2], rows=8, before=2, dtype=torch.float32),
         dict(counts=[5, 0], rows=9, before=1)]


@pytest.mark.parametrize("kw", CASES)
def test_everything_in_the_form_for_few_rows(kw):
    for wide in (47, 1):  # split and joined; a workgroup for a tile
        call = Call(**kw, lengths=(3000, 300) if wide > 1 else (64, 30))
        q = call.native("few")
        need = nv.lib().vl_attend_workspace_bytes(call.cache._ref, call.tokens, q)
        assert (need > 0) == (wide > 1)
        nv.check(nv.lib().vl_attend(call.cache._ref, call.tokens, q, nv.ptr(call.workspace(need)), need, nv.stream()))
        call.check()


def test_everything_in_the_form_for_many_rows():
    call = Call([300, 20], 400, heads=1, lengths=(5000, 300), before=30)
    q = call.native("many")
    need = nv.lib().vl_attend_workspace_bytes(call.cache._ref, call.tokens, q)
    assert need > 0
    nv.check(nv.lib().vl_attend(call.cache._ref, call.tokens, q, nv.ptr(call.workspace(need)), need, nv.stream()))
    assert (call.others(call.out) == MARK).all() and (call.others(call.lse) == MARK).all()
    want = dense(call.q, call.cache, call.table, call.lengths, call.at)
    check(call.out[call.mine], call.lse[call.mine], tuple(t[call.mine] for t in want), call.q.dtype, 64)


# blocks: scores in LDS and the choice in one launch, scores in the workspace and a launch more
@pytest.mark.parametrize("blocks", [47, 1100])
@pytest.mark.parametrize("kw", CASES)
def test_choice(kw, blocks):
    call = Call(**kw, blocks=blocks)
    (q, chosen) = (call.native(), call.list(4))
    need = nv.lib().vl_select_blocks_workspace_bytes(call.cache._ref, call.tokens, q, 4)
    assert (need > 0) == (blocks > 1024)
    nv.check(nv.lib().vl_select_blocks(call.cache._ref, call.tokens, q, 4, chosen.data_ptr(), nv.ptr(call.workspace(need)), need, nv.stream()))
    assert (call.others(chosen) == MARKED).all()
    want = ref.selection(call.q, call.cache, call.table, call.lengths, 4, call.at)
    assert torch.equal(chosen[call.mine].cpu(), want[call.mine])


@pytest.mark.parametrize("count", [3, 40])
@pytest.mark.parametrize("kw", CASES)
def test_lists(kw, count):
    """Lists of rows that belong to no sequence hold blocks that are there."""
    call = Call(**kw)
    (q, chosen) = (call.native(), call.list(count))
    chosen.copy_(torch.arange(count, device=DEV) % 5)
    chosen[:, :, 3:] = 2147483647
    need = nv.lib().vl_attend_blocks_workspace_bytes(call.cache._ref, call.tokens, q, count)
    assert (need > 0) == (count > 16)
    nv.check(nv.lib().vl_attend_blocks(call.cache._ref, call.tokens, q, chosen.data_ptr(), count, nv.ptr(call.workspace(need)), need, nv.stream()))
    call.check(chosen)


# rows x heads of 256 and more: in several launches; fewer: in one, or in several where one workgroup would read too much
@pytest.mark.parametrize("kw,blocks,alone", [(CASES[0], 47, True), (CASES[1], 47, True), (dict(counts=[100, 90], rows=300, before=20), 47, False),
                                             (CASES[2], 16_000, False)])
def test_choice_and_attention_over_it(kw, blocks, alone):
    call = Call(**kw, blocks=blocks)
    (q, chosen) = (call.native(), call.list(4))
    need = nv.lib().vl_attend_selected_workspace_bytes(call.cache._ref, call.tokens, q, 4)
    if alone:
        assert need == 0
    nv.check(nv.lib().vl_attend_selected(call.cache._ref, call.tokens, q, 4, chosen.data_ptr(), nv.ptr(call.workspace(need)), need, nv.stream()))
    assert (call.others(chosen) == MARKED).all()
    if blocks < 100:
        assert torch.equal(chosen[call.mine].cpu(), ref.selection(call.q, call.cache, call.table, call.lengths, 4, call.at)[call.mine])
    call.check(chosen)


def test_reading():
    """Rows of no sequence read as zeros, and not as what stands before or behind a sequence's."""
    call = Call([7, 5], 40, before=9)
    (k, v) = call.cache.read(call.table, call.lengths - 12, 40, call.at)
    assert not call.others(k).any() and not call.others(v).any()
    held = ref.Held(call.cache, call.table, call.lengths.tolist())
    for h in range(2):
        assert torch.equal(k[9:16, h].cpu().double(), held.k[0, h][2988:2995]) and torch.equal(v[16:21, h].cpu().double(), held.v[1, h][288:293])


def test_writing():
    call = Call([7, 5], 40, before=9)
    (gen, before) = (torch.Generator(device=DEV).manual_seed(1), [t.clone() for t in (call.cache.keys, call.cache.values)])
    x = torch.randn((2, 40, 2, 64), generator=gen, device=DEV).bfloat16()
    starts = call.lengths - 12
    call.cache.write(x[0], x[1], call.table, starts, call.at)
    (k, v) = call.cache.read(call.table, starts, 40, call.at, dtype=torch.float32)
    assert torch.equal(k[call.mine].cpu().double(), ref.rounded(x[0, call.mine])) and torch.equal(v[call.mine].cpu().double(), ref.rounded(x[1, call.mine]))
    # written as they were, the rows give back what the cache held: nothing else has changed
    was = attention.KVCache(before[0], call.cache.key_scales, before[1], call.cache.value_scales, call.cache.bounds, call.cache.bound_scales)
    for (now, then) in ((call.cache.keys, was.keys), (call.cache.values, was.values)):
        changed = (now != then).flatten(1).any(1).nonzero().flatten().tolist()
        touched = {int(call.table[b, i]) for (b, first, n) in ((0, 2988, 7), (1, 288, 5)) for i in range(first // 64, (first + n - 1) // 64 + 1)}
        assert set(changed) <= touched

"""Tree speculation operators on the CPU: the plain forms against independent restatements, and every refusal."""
import pytest
import torch

from antfly_b200.ops import attention as A
from antfly_b200.ops import tree as TR
from antfly_b200.runtime.kv_cache import BlockAllocator
from tests.helpers.tree_cases import Case, assert_close, random_trees

i32 = lambda v: torch.tensor(v, dtype=torch.int32)


def test_step_maps_equal_the_block_allocators_answers():
    page, max_blocks = 8, 16
    alloc = BlockAllocator(64, page)
    before, q = [5, 0, 17, 8], [3, 11, 0, 1]
    ids, slots, pos = [], [], []
    for s, (n, m) in enumerate(zip(before, q)):
        alloc.attach(s)
        alloc.append(s, n)
    for s, (n, m) in enumerate(zip(before, q)):
        slots += alloc.append(s, m).tolist()
        pos += range(n, n + m)
        ids += alloc.block_table(s).tolist()
    m = TR.step_maps(i32(before), i32(q), i32(ids), page, max_blocks, sum(q) + 2)
    assert m.slots.tolist() == slots + [-1, -1] and m.positions.tolist() == pos + [0, 0]
    assert m.q_starts.tolist() == [0, 3, 14, 14] and m.kv_lens.tolist() == [8, 11, 17, 9]
    assert m.logit_rows.tolist() == [2, 13, 13, 14]
    for s in range(4):
        t = alloc.block_table(s).tolist()
        assert m.block_tables[s].tolist() == t + [0] * (max_blocks - len(t))


def test_step_maps_of_a_tree_level_take_positions_from_depths():
    parents = i32([[-1, 0, 0, 1, 1, 2]])
    masks, depths = TR.tree_plan(parents)
    assert depths.tolist() == [[0, 1, 1, 2, 2, 2]]
    assert masks[0, :, 0].tolist() == [1, 3, 5, 0b1011, 0b10011, 0b100101]
    # the last three nodes are one level; the first three are in the cache already
    m = TR.step_maps(i32([10 + 3]), i32([3]), i32([4, 9]), 8, 4, 3, depths=depths, tree_lens=i32([6]), shift=i32([100]))
    assert m.positions.tolist() == [112, 112, 112] and m.slots.tolist() == [9 * 8 + 5, 9 * 8 + 6, 9 * 8 + 7]


def test_tree_plan_past_word_borders_and_short_trees():
    n = 70
    chain = torch.arange(-1, n - 1, dtype=torch.int32)[None]
    masks, depths = TR.tree_plan(chain.expand(2, n).contiguous(), i32([n, 33]))
    assert depths[0].tolist() == list(range(n)) and depths[1].tolist() == list(range(33)) + [0] * 37
    assert masks[0, 69].tolist() == [-1, -1, 0b111111] and masks[1, 32].tolist() == [-1, 1, 0]
    assert masks[1, 33:].abs().sum() == 0


def test_a_chain_is_causal_attention():
    c = Case([9, 0, 30], [5, 3, 1], 4, 2, 64, 8, seed=3)
    chain = torch.arange(-1, 4, dtype=torch.int32)[None].expand(3, 5).contiguous()
    c.masks, c.depths = TR.tree_plan(chain, c.q_lens)
    args, kw = c.args("cpu")
    got = TR.tree_attention(*args, **kw)
    want = A.paged_attention(c.q, c.k, c.v, c.tables, c.q_starts, c.q_lens, c.kv_lens, 5)
    torch.testing.assert_close(got.float(), want.float(), atol=1e-2, rtol=1e-2)
    assert_close(got, *c.exact())


def test_masked_values_never_enter_and_empty_rows_are_zero():
    c = Case([0, 20], [4, 4], 4, 2, 64, 8, seed=4)
    c.masks[0, 2] = 0                                             # sees nothing: no context, no node
    c.masks[1, 1] = 0b10
    exact, weighted = c.exact()
    other = int(c.tables[1, 22 // 8]) * 8 + 22 % 8                # node 2 of sequence 1: not an ancestor of node 1
    c.v.view(-1, 2, 64)[other] = float("nan")
    c.k.view(-1, 2, 64)[other] = float("inf")
    args, kw = c.args("cpu")
    got = TR.tree_attention(*args, **kw)
    assert (got[2] == 0).all()
    assert_close(got[:6], exact[:6], weighted[:6])


def test_accept_walks_to_the_lowest_agreeing_child_and_keeps_its_rows():
    parents = i32([[-1, 0, 0, 1, 2, 2], [-1, 0, 1, 2, 3, 4], [-1, 0, 0, 0, 0, 0]])
    tokens = i32([[1, 7, 7, 5, 6, 6], [1, 2, 3, 4, 5, 6], [1, 2, 3, 4, 5, 6]])
    target = i32([[7, 5, 6, 9, 9, 9], [2, 3, 4, 5, 6, 7], [9, 0, 0, 0, 0, 0]])
    k = torch.arange(2 * 4 * 8, dtype=torch.float32).view(2, 4, 8, 1, 1).repeat(1, 1, 1, 2, 4)
    v = -k
    slots = torch.stack([torch.arange(6) + 1, torch.arange(6) + 9, torch.arange(6) + 17]).int()
    kk, vv = k.clone(), v.clone()
    path, count, following = TR.tree_accept(tokens, parents, target, i32([6, 4, 6]), caches=[(kk, vv, slots)])
    assert path.tolist() == [[0, 1, 3, -1, -1, -1], [0, 1, 2, 3, -1, -1], [0, -1, -1, -1, -1, -1]]
    assert count.tolist() == [3, 4, 1] and following.tolist() == [9, 5, 9]
    want = k.clone()
    want.view(2, 32, -1)[:, 3] = k.view(2, 32, -1)[:, 4]          # node 3 becomes the tree's third row
    assert torch.equal(kk, want) and torch.equal(vv, -want)
    kk = k.clone()
    TR.tree_accept(tokens, parents, target, caches=[(kk, v.clone(), slots, 3)])
    assert torch.equal(kk, k)                                     # node 3 has no row in this cache


def test_refusals_name_what_is_wrong():
    c = Case([9], [3], 4, 2, 64, 8)
    args, kw = c.args("cpu")

    def call(at=None, value=None, **more):
        a = list(args)
        if at is not None:
            a[at] = value
        return TR.tree_attention(*a, **{**kw, **more})

    with pytest.raises(ValueError, match="q must be"):
        call(0, c.q[0])
    with pytest.raises(ValueError, match="caches of one shape"):
        call(2, c.v[:, :, :, :32])
    with pytest.raises(ValueError, match="caches of one shape"):
        call(1, c.k.half())
    with pytest.raises(ValueError, match="heads 3 over 2"):
        call(0, c.q[:, :3])
    with pytest.raises(ValueError, match="kv_lens must be int32"):
        call(6, c.kv_lens.long())
    with pytest.raises(ValueError, match="q_lens|q_starts"):
        call(4, i32([0, 1]))
    with pytest.raises(ValueError, match="masks must be"):
        call(7, torch.zeros((1, 3, 2), dtype=torch.int32))
    with pytest.raises(ValueError, match="masks must be"):
        call(7, torch.zeros((1, 300, 10), dtype=torch.int32))
    with pytest.raises(ValueError, match="window needs the nodes' depths"):
        call(window=4, depths=None)
    with pytest.raises(ValueError, match="not negative"):
        call(max_kv=-1)
    with pytest.raises(ValueError, match="out must be"):
        call(out=torch.zeros(3, 4, 64))
    with pytest.raises(ValueError, match="1 to 256 nodes"):
        TR.tree_plan(random_trees(1, 257, 0))
    with pytest.raises(ValueError, match="parents must be int32"):
        TR.tree_plan(random_trees(1, 7, 0).long())
    with pytest.raises(ValueError, match="lens must be"):
        TR.tree_plan(random_trees(2, 7, 0), i32([7]))
    with pytest.raises(ValueError, match="blocks must be"):
        TR.step_maps(i32([1]), i32([1]), torch.zeros(2), 8, 4, 1)
    with pytest.raises(ValueError, match="bad sizes"):
        TR.step_maps(i32([1]), i32([1]), i32([0]), 0, 4, 1)
    with pytest.raises(ValueError, match="depths must be"):
        TR.step_maps(i32([1]), i32([1]), i32([0]), 8, 4, 1, depths=i32([0]))
    t = random_trees(1, 4, 0)
    with pytest.raises(ValueError, match="target must be"):
        TR.tree_accept(t, t, t[:, :3])
    with pytest.raises(ValueError, match="at most two caches"):
        TR.tree_accept(t, t, t, caches=[()] * 3)
    k = torch.zeros(2, 3, 8, 2, 4)
    with pytest.raises(ValueError, match="slots must be"):
        TR.tree_accept(t, t, t, caches=[(k, k, i32([[0, 1]]))])
    with pytest.raises(ValueError, match="contiguous"):
        TR.tree_accept(t, t, t, caches=[(k[:, :2], k[:, :2], t)])


@pytest.mark.parametrize("scale", [0.0, -0.125, float("nan"), float("inf"), -float("inf"), 1e-8, 1e5])
def test_scales_that_are_not_positive_numbers_are_refused(scale):
    c = Case([9, 70], [3, 2], 4, 2, 64, 8)
    args, kw = c.args("cpu")
    with pytest.raises(ValueError, match="scale must be a positive number"):
        TR.tree_attention(*args, scale=scale, **kw)


@pytest.mark.parametrize("scale", [1e-7, 1.0, 1e4])
def test_scales_at_the_ends_of_their_range(scale):
    c = Case([9, 70], [3, 2], 4, 2, 64, 8)
    args, kw = c.args("cpu")
    assert torch.isfinite(TR.tree_attention(*args, scale=scale, **kw)).all()


def test_codec_caches_ask_nothing_of_table_entries_behind_the_last_key():
    from antfly_b200.ops.kv_quant import CodecCache

    c = Case([9, 30], [3, 2], 4, 2, 64, 8, seed=6)
    k, v = (CodecCache("int8", 1, c.k.shape[0], 8, 2, 64, "cpu", value=x) for x in (False, True))
    at = torch.arange(c.k.shape[0] * 8, dtype=torch.int32)
    k[0].write(at, c.k.view(-1, 2, 64))
    v[0].write(at, c.v.view(-1, 2, 64))
    args, kw = c.args("cpu")
    want = TR.tree_attention(args[0], k[0], v[0], *args[3:], **kw)
    for odd in (99999, 1 << 30, -5):
        tables = torch.nn.functional.pad(args[3], (0, 2), value=odd)
        tables[0, 2:] = odd                                       # 12 keys: two pages
        assert torch.equal(TR.tree_attention(args[0], k[0], v[0], tables, *args[4:], **{**kw, "max_kv": 0}), want)
    tables = args[3].clone()
    tables[0, 1] = 1 << 28                                        # times the page size, no id of 32 bits
    with pytest.raises(IndexError):
        TR.tree_attention(args[0], k[0], v[0], tables, *args[4:], **kw)


def test_caches_that_share_memory_are_refused():
    """Their rows would be moved twice, the second time from where the first move put another node's."""
    t = i32([[-1, 0, 0, 2, 3]])
    slots = i32([[0, 1, 2, 3, 4]])
    k, v = torch.zeros(2, 3, 8, 2, 4), torch.zeros(2, 3, 8, 2, 4)
    for caches in ([(k, k, slots)], [(k, v, slots), (v, k, slots)], [(k, v, slots), (k, v, slots)],
                   [(k, v, slots), (k[1:], torch.zeros(1, 3, 8, 2, 4), slots)]):
        with pytest.raises(ValueError, match="share memory"):
            TR.tree_accept(t, t, t, caches=caches)
    both = torch.arange(2 * 2 * 24 * 8, dtype=torch.float32).view(2, 2, 3, 8, 2, 4)      # two halves of one tensor do not
    TR.tree_accept(t, t, t, caches=[(both[0], both[1], slots)])

"""accept_tree on the GPU against a walk over each tree."""

import pytest
import torch

from kv_reference import accept

from dspine_b200 import accept as A
from dspine_b200.attention import tree_mask

pytestmark = pytest.mark.gpu


def _tree(g, n, wide):
    parents = [-1]
    for i in range(1, n):
        parents.append(int(torch.randint(0, i, (1,), generator=g)) if wide else max(0, i - 1 - int(torch.randint(0, 3, (1,), generator=g))))
    return parents


def _masks(parents):
    return tree_mask(torch.tensor(parents, dtype=torch.int64)) if parents else torch.zeros(0, dtype=torch.int64)


def _batch(widths, seed, wide, vocab=3):
    g = torch.Generator().manual_seed(seed)
    trees = [_tree(g, n, wide) if n else [] for n in widths]
    n = sum(widths)
    tokens = torch.randint(0, vocab, (n,), generator=g)
    top1 = torch.randint(0, vocab, (n,), generator=g)
    return trees, tokens, top1, torch.cat([_masks(t) for t in trees]) if n else torch.zeros(0, dtype=torch.int64)


def _expect(trees, tokens, top1, slots, prefix, width):
    want = {k: [] for k in ("accept", "commit", "bonus", "output", "path", "kept_slots", "new_seq")}
    lo = 0
    for b, t in enumerate(trees):
        n = len(t)
        path, out, bonus = accept(tokens[lo:lo + n].tolist(), top1[lo:lo + n].tolist(), t)
        c = len(path)
        want["accept"].append(max(c - 1, 0))
        want["commit"].append(c)
        want["bonus"].append(bonus)
        want["output"].append(out + [0] * (width - c))
        want["path"].append(path + [-1] * (width - c))
        want["kept_slots"].append([int(slots[lo + i]) for i in path] + [-1] * (width - c))
        want["new_seq"].append(int(prefix[b]) + c)
        lo += n
    return want


def _same(got, want):
    for name, w in want.items():
        g = getattr(got, name)
        assert g.cpu().tolist() == w, name


@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("widths", [[1], [2, 1], [64], [16] * 5, [33, 0, 64, 1, 32, 31, 7], [0, 0], list(range(1, 65))])
def test_ragged_trees(widths, wide):
    for seed in range(4):
        trees, tokens, top1, mask = _batch(widths, seed, wide)
        slots = torch.randperm(4000)[:sum(widths)].int()
        prefix = torch.arange(len(widths), dtype=torch.int32) * 10
        starts = torch.tensor([0] + widths).cumsum(0).int()
        got = A.accept_tree(tokens.cuda(), top1.cuda(), mask.cuda(), q_indptr=starts.cuda(), prefix_lens=prefix.cuda(),
                            slots=slots.cuda())
        _same(got, _expect(trees, tokens, top1, slots, prefix, 64))


@pytest.mark.parametrize("nodes,width", [(1, 1), (16, 16), (16, 20), (64, 64), (5, 64)])
def test_uniform_trees_without_slots(nodes, width):
    trees, tokens, top1, mask = _batch([nodes] * 9, nodes, False, vocab=2)
    shape = (9, nodes)
    got = A.accept_tree(tokens.view(shape).cuda(), top1.view(shape).cuda(), mask.view(shape).cuda(), width=width)
    want = _expect(trees, tokens, top1, torch.zeros(9 * nodes), torch.zeros(9), width)
    del want["kept_slots"]
    assert got.kept_slots is None
    _same(got, want)


def test_a_chain_is_the_chain_accept():
    """On chains of 16 tree acceptance is accept_greedy."""
    g = torch.Generator().manual_seed(5)
    B = 40
    tokens, top1 = torch.randint(0, 2, (B, 16), generator=g).cuda(), torch.randint(0, 2, (B, 16), generator=g).cuda()
    mask = tree_mask(torch.arange(-1, 15)).expand(B, 16).contiguous().cuda()
    got = A.accept_tree(tokens, top1, mask)
    accept, commit, bonus, output, new_seq = A.accept_greedy(tokens, top1, torch.full((B,), 16, dtype=torch.int32, device="cuda"))
    for x, y in ((got.accept, accept), (got.commit, commit), (got.bonus, bonus), (got.new_seq, new_seq)):
        assert torch.equal(x, y)
    for b in range(B):
        assert torch.equal(got.output[b, :int(commit[b])], output[b, :int(commit[b])])


def test_masks_that_are_no_trees_and_equal_siblings():
    """Bits above a node are not read, its own bit counts as set, a node without the root above it is never
    accepted, and of equally deep nodes the first one wins."""
    tokens = torch.tensor([[9, 5, 5, 7, 7, 1]]).cuda()
    top1 = torch.tensor([[5, 7, 7, 1, 1, 3]]).cuda()
    #        root, child of 0, child of 0, child of 1, child of 2, no parent
    mask = torch.tensor([[0, 1, 0b101, 0b1011, 0b10101 | (1 << 40), 0]]).cuda()
    got = A.accept_tree(tokens, top1, mask)
    assert got.path[0].tolist() == [0, 1, 3, -1, -1, -1] and int(got.bonus[0]) == 1
    assert got.output[0].tolist() == [5, 7, 1, 0, 0, 0] and int(got.accept[0]) == 2


def test_only_the_first_rows_are_looked_at_and_bad_offsets_stay_inside():
    trees, tokens, top1, mask = _batch([64], 3, False, vocab=1)    # every node agrees
    got = A.accept_tree(tokens.cuda(), top1.cuda(), mask.cuda(), q_indptr=torch.tensor([0, 64], dtype=torch.int32).cuda(), width=7)
    want = _expect([trees[0][:7]], tokens[:7], top1[:7], torch.zeros(7), torch.zeros(1), 7)
    assert got.path.cpu().tolist() == want["path"]
    bad = torch.tensor([-5, 200, 10, 64], dtype=torch.int32).cuda()   # read as [0, 64), none, [10, 64)
    got = A.accept_tree(tokens.cuda(), top1.cuda(), mask.cuda(), q_indptr=bad)
    assert got.commit[0] > 0 and int(got.commit[1]) == 0 and int(got.bonus[1]) == -1


def test_empty_batches_and_given_outputs():
    z = torch.zeros(0, dtype=torch.int64, device="cuda")
    got = A.accept_tree(z, z, z, q_indptr=torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert got.accept.numel() == 0
    trees, tokens, top1, mask = _batch([8] * 3, 4, True)
    out = A.TreeAccept.allocate(3, 8, "cuda", slots=False)
    shape = (3, 8)
    assert A.accept_tree(tokens.view(shape).cuda(), top1.view(shape).cuda(), mask.view(shape).cuda(), outputs=out) is out
    want = _expect(trees, tokens, top1, torch.zeros(24), torch.zeros(3), 8)
    del want["kept_slots"]
    _same(out, want)

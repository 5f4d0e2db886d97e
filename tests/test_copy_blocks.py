"""Copies of cache blocks, forks of sequences that share blocks, and caches given another size: the
bookkeeping on the host's tensors (no GPU), and the copying kernel against plain indexing (bit for bit: it
computes nothing)."""

import numpy as np
import pytest
import torch

from semantic_aware_adaptive_kv_cache_precision_b200 import ops
from semantic_aware_adaptive_kv_cache_precision_b200.cache import (BLOCK, CacheFull, KVNeed, MultiNeed, SequenceCache,
                                                                    StateNeed)
from semantic_aware_adaptive_kv_cache_precision_b200.ops import KernelError

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def make(device, max_tokens=20 * BLOCK, window=None, keep_first=0, state=True, max_positions=1024, **how):
    needs = [KVNeed(2, 16), KVNeed(2, 16), KVNeed(1, 32, window, keep_first=keep_first),
             MultiNeed((KVNeed(1, 8, value_dim=0), StateNeed((5,), "int32")))]
    if state:
        needs.append(StateNeed((3, 4), "float32"))
    return SequenceCache(needs, max_tokens, max_positions, torch.float32, device, **how)


def fill(cache, slot, length, seed):
    """Feed a sequence up to `length` positions and write recognisable numbers everywhere it owns."""
    rng = np.random.default_rng(seed)
    start = int(cache.lengths[slot])
    cache.reserve([slot], [length])
    for group in cache.groups:
        for c in range(start // BLOCK, -(-length // BLOCK)):
            block = int(group.tables[slot, c])
            for t in group.tensors:
                a, z = max(start, c * BLOCK) - c * BLOCK, min(length, (c + 1) * BLOCK) - c * BLOCK
                t[:, block, :, a:z] = torch.as_tensor(rng.standard_normal(t[:, block, :, a:z].shape),
                                                      dtype=t.dtype, device=t.device)
    for state in cache.states.values():
        state[slot] = torch.as_tensor(rng.integers(1, 100, state[slot].shape)).to(state)
    cache.advance([slot], [length])


def content(cache, slot):
    """What a sequence has: per group and tensor the filled positions it still holds, and its state."""
    n = int(cache.lengths[slot])
    out = []
    for group in cache.groups:
        row = group.tables[slot]
        for t in group.tensors:
            for c in range(-(-n // BLOCK)):
                if row[c] >= 0:
                    out.append(t[:, int(row[c]), :, :min(BLOCK, n - c * BLOCK)].clone())
    return out + [s[slot].clone() for s in cache.states.values()]


def same(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("length", [0, 1, 63, 64, 65, 128, 200])
def test_a_fork_has_what_its_parent_has_and_goes_its_own_way(device, length):
    cache = make(device)
    (a,) = cache.open(1)
    fill(cache, a, length, 1)
    held = cache.groups[0].pool.held
    new = cache.fork(a, 3)
    cache.check()
    assert len(new) == 3 and a not in new
    # whole blocks are shared, the partly filled one is each sequence's own
    assert cache.groups[0].pool.held == held + (3 if length % BLOCK else 0)
    assert cache.shares_blocks == (length >= BLOCK)
    before = content(cache, a)
    assert all(cache.lengths[s] == length and same(content(cache, s), before) for s in new)
    fill(cache, new[0], length + 70, 2)
    fill(cache, a, length + 1, 3)
    cache.check()
    assert same(content(cache, new[1]), before) and same(content(cache, new[2]), before)
    mine = content(cache, new[0])
    cache.close([a, new[1]])
    cache.check()
    assert same(content(cache, new[0]), mine) and same(content(cache, new[2]), before)
    cache.close([new[0], new[2]])
    cache.check()
    assert not cache.shares_blocks and all(g.pool.held == 0 for g in cache.groups)


@pytest.mark.parametrize("device", DEVICES)
def test_forks_of_forks_and_poisoned_blocks(device):
    cache = make(device, poison_freed=True)
    (a,) = cache.open(1)
    fill(cache, a, 130, 1)
    (b,) = cache.fork(a)
    fill(cache, b, 300, 2)
    c, d = cache.fork(b, 2)
    want = content(cache, b)
    cache.close([a])
    cache.close([b])
    cache.check()
    assert same(content(cache, c), want) and same(content(cache, d), want)
    assert not any(x.isnan().any() for x in want if x.is_floating_point())
    cache.close([c])
    assert cache.shares_blocks is False and same(content(cache, d), want)
    cache.close([d])
    cache.check()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("keep_first", [0, 70])
def test_windows_give_back_shared_blocks_once(device, keep_first):
    cache = make(device, window=100, keep_first=keep_first)
    (a,) = cache.open(1)
    fill(cache, a, 200, 1)
    (b,) = cache.fork(a)
    cache.check()
    want = content(cache, b)
    fill(cache, a, 450, 2)             # the window's group gives back what a no longer sees
    cache.check()
    assert same(content(cache, b), want)
    fill(cache, b, 451, 3)
    cache.check()
    (c,) = cache.fork(b)
    assert same(content(cache, c), content(cache, b))
    cache.close([a, b, c])
    cache.check()


@pytest.mark.parametrize("device", DEVICES)
def test_a_fork_is_all_or_nothing(device):
    cache = make(device, max_tokens=4 * BLOCK, max_slots=4)
    (a,) = cache.open(1)
    fill(cache, a, 100, 1)
    with pytest.raises(CacheFull):
        cache.fork(a, 3)                        # two free blocks for three last blocks
    with pytest.raises(CacheFull):
        cache.fork(a, 4)
    cache.check()
    assert cache.slots.held == 1 and cache.groups[0].pool.held == 2 and not cache.shares_blocks
    assert cache.fork(a, 0) == []
    with pytest.raises(ValueError):
        cache.fork(a, -1)
    with pytest.raises(RuntimeError, match="not held"):
        cache.fork(3)
    assert len(cache.fork(a, 2)) == 2
    cache.check()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("size", [6 * BLOCK, 6 * BLOCK - 1, 20 * BLOCK, 40 * BLOCK])
def test_a_cache_of_another_size_has_the_same_sequences(device, size):
    cache = make(device, window=80)
    a, b, gone = cache.open(3)
    fill(cache, gone, 190, 1)
    fill(cache, a, 150, 2)
    (c,) = cache.fork(a)
    fill(cache, c, 170, 3)
    fill(cache, b, 64, 4)
    cache.close([gone])
    before = [content(cache, s) for s in (a, b, c)]
    cache.resize(size)
    cache.check()
    assert cache.blocks == -(-size // BLOCK) and cache.max_tokens == cache.blocks * BLOCK
    assert cache.groups[0].keys.shape[1] == cache.blocks and cache.shares_blocks
    assert all(same(content(cache, s), x) for s, x in zip((a, b, c), before))
    # held blocks lie at the front, and the sequences go on
    assert all(sorted(g.pool._held) == list(range(g.pool.held)) for g in cache.groups)
    fill(cache, b, 100, 5)
    cache.check()
    cache.close([a, b, c])
    cache.check()
    assert cache.max_seq_len == min(1024, cache.max_tokens)


@pytest.mark.parametrize("device", DEVICES)
def test_a_larger_cache_may_have_more_slots(device):
    cache = make(device, max_tokens=3 * BLOCK, max_slots=2, window=80)
    a, b = cache.open(2)
    fill(cache, a, 70, 1)
    fill(cache, b, 10, 2)
    before = [content(cache, s) for s in (a, b)]
    cache.resize(30 * BLOCK, 7)
    cache.check()
    assert cache.max_slots == 7 and all(t.shape[0] == 7 for t in cache.states.values())
    assert all(same(content(cache, s), x) for s, x in zip((a, b), before))
    new = cache.fork(a, 5)
    assert new == [2, 3, 4, 5, 6] and all(same(content(cache, s), before[0]) for s in new)
    with pytest.raises(CacheFull):
        cache.open(1)
    cache.close(new + [a, b])
    cache.resize(BLOCK, 1)                       # slots never become fewer
    cache.check()
    assert cache.max_slots == 7 and cache.slots.free == 7


@pytest.mark.parametrize("device", DEVICES)
def test_a_size_that_does_not_hold_the_sequences_is_refused(device):
    cache = make(device)
    a, b = cache.open(2)
    fill(cache, a, 200, 1)
    fill(cache, b, 300, 2)
    before = [content(cache, s) for s in (a, b)]
    for size in (8 * BLOCK, 4 * BLOCK):             # nine blocks are held; the longer sequence has five
        with pytest.raises(CacheFull, match="nothing was changed"):
            cache.resize(size)
    with pytest.raises(ValueError):
        cache.resize(0)
    cache.check()
    assert cache.blocks == 20 and all(same(content(cache, s), x) for s, x in zip((a, b), before))
    cache.resize(9 * BLOCK)
    cache.check()
    assert all(same(content(cache, s), x) for s, x in zip((a, b), before))


# -- the kernel --------------------------------------------------------------------------

def test_refusals():
    t = torch.zeros(2, 6, 1, 8, 4)
    copy = ops.copy_blocks
    for args, how in ((([t], [0], [6]), {}), (([t], [-1], [1]), {}), (([t], [0, 1], [2]), {}),
                      (([t], [0, 1], [2, 2]), {}), (([t], [0, 1], [2, 1]), {}), (([t], [0], [1]), {"rows": 0}),
                      (([t], [0], [1]), {"rows": 9}), (([t], [0], [1]), {"axis": 2}),
                      (([t[0]], [0], [1]), {"rows": 3}), (([t], [0], [1]), {"into": []}),
                      (([t], [0], [1]), {"into": [t.double()]}), (([t], [0], [1]), {"into": [t[:, :, :, :7]]}),
                      (([t], [0], [1]), {"into": [t]}), (([t[:, ::2]], [0], [1]), {}),
                      (([t, torch.zeros(2, 5, 1, 8, 4)], [0], [1]), {}), (([t, t], [0], [1]), {}),
                      (([t], [0], [3]), {"into": [torch.zeros(2, 3, 1, 8, 4)]})):
        with pytest.raises(KernelError):
            copy(*args, **how)
    with pytest.raises(KernelError, match="CUDA device only"):
        copy([t], [0], [1])


SHAPES = [(1, 9, 1, 64, 1), (3, 9, 2, 64, 16), (2, 9, 3, 64, 5), (1, 9, 1, 64, 2), (4, 9, 2, 64, 48), (2, 9, 2, 64, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.int32, torch.uint8])
@pytest.mark.parametrize("rows", [None, 1, 37, 64])
@pytest.mark.parametrize("fresh", [False, True])
def test_blocks_against_indexing(dtype, rows, fresh):
    g = torch.Generator().manual_seed(3)
    tensors = [torch.randint(0, 200, s, generator=g).to(dtype).cuda() for s in SHAPES]
    src, dst = [4, 4, 0, 8], [1, 2, 7, 3]
    into = [torch.randint(0, 200, (s[0], 11) + s[2:], generator=g).to(dtype).cuda() for s in SHAPES] if fresh else None
    want = [t.clone() for t in (into or tensors)]
    for w, t in zip(want, tensors):
        w[:, dst, :, :rows] = t[:, src, :, :rows]
    ops.copy_blocks(tensors, src, dst, into=into, rows=rows)
    assert all(torch.equal(a, b) for a, b in zip(into or tensors, want))


@pytest.mark.gpu
def test_states_many_pairs_and_nothing():
    g = torch.Generator().manual_seed(4)
    states = [torch.randn((5000,) + s, generator=g).cuda() for s in ((3, 4), (7,), ())]
    order = torch.randperm(5000, generator=g).tolist()
    src, dst = order[:2300], order[2300:4600]           # three launches
    want = [s.clone() for s in states]
    for w, s in zip(want, states):
        w[dst] = s[src]
    ops.copy_blocks(states, src, dst, axis=0)
    assert all(torch.equal(a, b) for a, b in zip(states, want))
    ops.copy_blocks(states, [], [], axis=0)
    ops.copy_blocks([], [], [])
    many = [torch.randn((2, 4, 1, 64, 8), generator=g).cuda() for _ in range(40)]       # more tensors than a launch takes
    want = [m.clone() for m in many]
    for w in want:
        w[:, 3] = w[:, 0]
    ops.copy_blocks(many, [0], [3])
    assert all(torch.equal(a, b) for a, b in zip(many, want))


@pytest.mark.gpu
def test_copies_past_four_gigabytes_and_captured():
    t = torch.zeros((1, 5000, 4, 64, 1024), dtype=torch.bfloat16, device="cuda")        # 2.6 GB, 512 KB a block
    assert t.numel() * 2 > 1 << 31
    t[0, 4999] = torch.randn(4, 64, 1024).to(t)
    other = torch.zeros((1, 9000, 4, 64, 1024), dtype=torch.bfloat16, device="cuda")
    ops.copy_blocks([t], [4999, 4999], [8999, 0], into=[other])
    assert torch.equal(other[0, 8999], t[0, 4999]) and torch.equal(other[0, 0], t[0, 4999])
    assert not other[0, 1].any() and not other[0, 8998].any()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.copy_blocks([t], [4999], [17], rows=5)
    assert not t[0, 17].any()
    t[0, 4999] += 1
    graph.replay()
    assert torch.equal(t[0, 17, :, :5], t[0, 4999, :, :5]) and not t[0, 17, :, 5:].any()


@pytest.mark.gpu
def test_tensors_of_no_size_beside_others():
    g = torch.Generator().manual_seed(6)
    states = [torch.randn((8,) + s, generator=g).cuda() for s in ((0, 7), (3, 4), (2, 0), (5,))]
    want = [s.clone() for s in states]
    for w in want:
        w[[1, 6]] = w[[0, 3]]
    ops.copy_blocks(states, [0, 3], [1, 6], axis=0)
    assert all(torch.equal(a, b) for a, b in zip(states, want))
    pools = [torch.randn(s, generator=g).cuda() for s in ((0, 8, 2, 64, 4), (3, 8, 2, 64, 4), (1, 8, 2, 64, 0))]
    want = [p.clone() for p in pools]
    want[1][:, 2, :, :9] = want[1][:, 5, :, :9]
    ops.copy_blocks(pools, [5], [2], rows=9)
    assert all(torch.equal(a, b) for a, b in zip(pools, want))
    ops.copy_blocks([pools[0], pools[2]], [5], [2])                # nothing at all to copy
    for bad in (lambda: ops.copy_blocks(pools, [8], [2]), lambda: ops.copy_blocks([pools[0]], [0], [8]),
                lambda: ops.copy_blocks([pools[0], states[0]], [0], [1])):
        with pytest.raises(KernelError):
            bad()


@pytest.mark.parametrize("device", DEVICES)
def test_state_of_no_size_keeps_no_other_state_from_moving(device):
    """A mixer whose convolution has one tap keeps no inputs beside its recurrent state."""
    needs = [KVNeed(2, 16), MultiNeed((StateNeed((0, 6), "float32"), StateNeed((2, 3), "float32"))), StateNeed((4,), "int32")]
    cache = SequenceCache(needs, 6 * BLOCK, 1024, torch.float32, device, max_slots=3)
    (a,) = cache.open(1)
    fill(cache, a, 70, 1)
    want = content(cache, a)
    (b,) = cache.fork(a)
    assert same(content(cache, b), want)
    cache.resize(12 * BLOCK, 9)
    cache.check()
    assert same(content(cache, a), want) and same(content(cache, b), want)


def test_block_numbers_are_whole_and_read_as_often_as_needed():
    t = torch.zeros(2, 6, 1, 8, 4)
    for src, dst in (([1.7], [2]), ([1], [2.0]), (["1"], [2]), ([1], [None]), ([2 ** 70], [1]),
                     (np.array([1.0]), np.array([2])), (torch.tensor([1.5]), [2])):
        with pytest.raises(KernelError, match="whole numbers"):
            ops.copy_blocks([t], src, dst)
    for src, dst in ((iter([1]), iter([2 ** 40])), (iter([-1]), [2]), (np.array([1]), np.array([6])),
                     (torch.tensor([7]), [2])):
        with pytest.raises(KernelError, match="must lie in"):
            ops.copy_blocks([t], src, dst)
    for src, dst in ((iter([1]), iter([2])), (np.array([1]), np.array([2], dtype=np.int16)), (torch.tensor([1]), range(2, 3))):
        with pytest.raises(KernelError, match="CUDA device only"):
            ops.copy_blocks([t], src, dst)

"""Decode attention over blocks that several sequences list: the plan (no GPU), and the kernel against a
float64 softmax over each sequence's own positions."""

import math

import numpy as np
import pytest
import torch

from semantic_aware_adaptive_kv_cache_precision_b200 import ops
from semantic_aware_adaptive_kv_cache_precision_b200.ops import KernelError
from semantic_aware_adaptive_kv_cache_precision_b200.ops.shared import common_runs, choose_piece

BLOCK = 64


def lists_of(prompts):
    """Block lists as forks make them: `prompts` [(shared, [(second common piece, tail)])]. Returns (tables,
    lengths, blocks)."""
    lists, lengths, taken = [], [], 0
    for shared, rows in prompts:
        common = list(range(taken, taken + shared // BLOCK))
        taken += len(common)
        branches = {}
        for again, tail in rows:
            at, mine = shared + again, list(common)
            if again:
                if again not in branches:
                    n = at // BLOCK - len(common)
                    branches[again] = list(range(taken, taken + n))
                    taken += n
                mine += branches[again]
            n = -(-(at + tail) // BLOCK) - len(mine)
            mine += range(taken, taken + n)
            taken += n
            lists.append(mine)
            lengths.append(at + tail)
    width = max(max(map(len, lists)), 1) + 1
    return np.array([x + [-1] * (width - len(x)) for x in lists]), np.array(lengths), taken


def covered(plan, tables, reach):
    """Every column of every sequence exactly once, by a unit that reads the sequence's own block; every
    partial written once, and among the sequence's own. Returns the blocks read."""
    w = np.asarray(plan.words)
    count, read = len(reach), []
    first = w[plan.first_at:plan.first_at + count + 1]
    seen, partials = [set() for _ in reach], set()
    group = plan.heads // plan.kv_heads
    heads_of = {}
    assert w[0] == plan.units <= plan.unit_capacity and w[1] == count
    for unit in w[plan.unit_at:plan.unit_at + 8 * plan.units].reshape(-1, 8):
        row, c0, n, begin, first_row, rows = unit[:6]
        assert n > 0 and 0 < rows <= 128 and 0 <= first_row < group
        for r in range(first_row, first_row + rows):
            b, p = w[plan.member_at + 2 * (begin + r // group):][:2]
            assert first[b] <= p < first[b + 1] <= plan.partials
            heads_of.setdefault((b, p), []).append(r % group)
            if r % group == 0:
                assert p not in partials
                partials.add(p)
                for c in range(c0, c0 + n):
                    assert c not in seen[b] and tables[b, c] == tables[row, c]
                    seen[b].add(c)
        read += [(row, c) for c in range(c0, c0 + n)]
    assert len(partials) == first[-1] and all(sorted(h) == list(range(group)) for h in heads_of.values())
    assert all(s == set(range(-(-int(r) // BLOCK))) for s, r in zip(seen, reach))
    return read


CASES = {
    "one": [(0, [(0, 1)])],
    "alone": [(0, [(0, 700)]), (0, [(0, 65)]), (0, [(0, 64)])],
    "forks": [(1000, [(0, 7), (0, 60), (0, 200), (0, 1)])],
    "whole blocks": [(128, [(0, 64), (0, 1), (0, 130)])],
    "tree": [(640, [(0, 5), (100, 9), (100, 80), (300, 1), (300, 64)]), (70, [(0, 3), (64, 4), (64, 5)])],
    "many": [(900, [(0, 1 + 3 * i) for i in range(40)])],
    "empty": [(0, [(0, 0)]), (200, [(0, 1), (0, 2)]), (0, [(0, 0)])],
}


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("heads, kv_heads", [(12, 2), (8, 8), (16, 1)])
@pytest.mark.parametrize("slots", [1, 40, 296])
def test_a_plan_reads_every_column_once(name, heads, kv_heads, slots):
    tables, lengths, blocks = lists_of(CASES[name])
    plan = ops.plan_shared(tables, lengths, heads, kv_heads, slots=slots)
    read = covered(plan, tables, lengths)
    if heads == 8:                                   # (all rows fit a unit: nothing is read twice)
        assert len({tables[r, c] for r, c in read}) == len(read) == len({b for b in tables.reshape(-1) if b >= 0})
    grown = np.minimum(lengths + 100, tables.shape[1] * BLOCK)
    for roomy in (False, True):
        covered(ops.plan_shared(tables, lengths, heads, kv_heads, slots=slots, reach=grown, roomy=roomy), tables, grown)


def test_plans_of_any_lists():
    rng = np.random.default_rng(0)
    for _ in range(60):
        count, width = int(rng.integers(1, 9)), int(rng.integers(1, 12))
        tables = rng.integers(0, 6, (count, width))            # the same blocks anywhere, twice in one list too
        lengths = rng.integers(0, width * BLOCK + 1, count)
        covered(ops.plan_shared(tables, lengths, 4, 2, slots=int(rng.integers(1, 30))), tables, lengths)
    covered(ops.plan_shared(np.zeros((0, 3), int), [], 4, 2, slots=8), np.zeros((0, 3), int), [])


def test_a_last_block_that_is_not_filled_is_nobody_elses():
    tables = np.array([[3, 4], [3, 4]])
    assert sorted(common_runs(tables, np.array([100, 128]), np.array([100, 128]))) == \
        [((0,), 1, 2), ((0, 1), 0, 1), ((1,), 1, 2)]


def test_pieces_fill_the_slots():
    runs = [(tuple(range(64)), 0, 500)] + [((b,), 500, 508) for b in range(64)]
    piece = choose_piece(runs, 6, 2, 296)
    assert 8 <= piece <= 40
    # many short tails do not make the prompts' pieces long
    runs = [(tuple(range(6 * p, 6 * p + 6)), 0, 374) for p in range(5)] + [((b,), 374, 380) for b in range(30)]
    assert choose_piece(runs, 5, 8, 296) <= 100
    assert choose_piece([((0,), 0, 1)], 6, 2, 296) == 1 and choose_piece([((0,), 0, 400)], 1, 1, 1) >= 100


def test_refusals():
    tables, lengths, _ = lists_of(CASES["forks"])
    for args in ((tables[:2], lengths, 12, 2), (tables, lengths, 12, 5), (tables, lengths, 0, 1),
                 (tables, -lengths, 12, 2), (tables, lengths + 5000, 12, 2), (tables, lengths, 130, 2),
                 (np.full_like(tables, -1), lengths, 12, 2), (tables[0], lengths, 12, 2)):
        with pytest.raises(KernelError):
            ops.plan_shared(*args, slots=8)
    with pytest.raises(KernelError):
        ops.plan_shared(tables, lengths, 12, 2, slots=8, reach=lengths - 1)
    plan = ops.plan_shared(tables, lengths, 12, 2, slots=8)
    plan = plan.on(torch.from_numpy(plan.words))
    b, width = tables.shape
    good = dict(qkv=torch.zeros(b, 12 * 64, dtype=torch.bfloat16), k_cache=torch.zeros(99, 2, 64, 64, dtype=torch.bfloat16),
                v_cache=torch.zeros(99, 2, 64, 64, dtype=torch.bfloat16),
                seq_lens=torch.zeros(b, dtype=torch.int32), block_table=torch.zeros(b, width, dtype=torch.int32),
                plan=plan, heads=12, kv_heads=2, head_dim=64, scale=1.0)
    for bad in (dict(qkv=good["qkv"].float()), dict(qkv=good["qkv"][:, :700]), dict(qkv=good["qkv"][:2]),
                dict(head_dim=128), dict(head_dim=48), dict(kv_heads=3), dict(heads=24), dict(heads=8),
                dict(seq_lens=good["seq_lens"].long()), dict(block_table=good["block_table"][:, 1:].contiguous()),
                dict(block_table=good["block_table"].t().contiguous().t()), dict(v_cache=good["v_cache"][:, :1]),
                dict(k_cache=good["k_cache"][:5]), {}):
        with pytest.raises(KernelError):
            ops.shared_decode_attention(**{**good, **bad})


def run(prompts, heads, kv_heads, d, seed=0, slots=None, poison=True, plan_at=None, q_pad=0):
    """(kernel's output, float64 reference, bound) of the sequences of `prompts`."""
    tables, lengths, blocks = lists_of(prompts)
    g = torch.Generator(device="cuda").manual_seed(seed)
    pool = blocks + 2
    order = np.random.default_rng(seed).permutation(pool)
    placed = np.where(tables >= 0, order[np.maximum(tables, 0)], -1).astype(np.int32)
    k = torch.randn((pool, kv_heads, BLOCK, d), generator=g, device="cuda").to(torch.bfloat16)
    v = torch.randn((pool, kv_heads, BLOCK, d), generator=g, device="cuda").to(torch.bfloat16)
    if poison:              # rows behind a sequence's end, and blocks nobody lists, hold what must not be read
        used = torch.zeros(pool, BLOCK, dtype=torch.bool)
        for row, n in zip(placed, lengths):
            for c in range(-(-int(n) // BLOCK)):
                used[row[c], :min(BLOCK, int(n) - c * BLOCK)] = True
        bad = ~used.cuda()[:, None, :, None].expand_as(k)
        k.masked_fill_(bad, math.nan)
        v.masked_fill_(bad, math.inf)
    b = len(lengths)
    q = torch.randn((b, heads * d + q_pad), generator=g, device="cuda").mul_(1.5).to(torch.bfloat16)
    scale = d ** -0.5
    at = lengths if plan_at is None else np.minimum(lengths, plan_at)
    plan = ops.plan_shared(placed, at, heads, kv_heads, device="cuda", slots=slots, reach=lengths)
    out = ops.shared_decode_attention(q, k, v, torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                                      torch.from_numpy(placed).cuda(), plan, heads, kv_heads, d, scale)
    ref = torch.zeros(b, heads, d, dtype=torch.float64)
    spread = torch.zeros_like(ref)
    group = heads // kv_heads
    for i, n in enumerate(lengths):
        if n == 0:
            continue
        mine = torch.from_numpy(placed[i, :-(-int(n) // BLOCK)]).long().cuda()
        keys = k[mine].permute(1, 0, 2, 3).reshape(kv_heads, -1, d)[:, :n].double()
        vals = v[mine].permute(1, 0, 2, 3).reshape(kv_heads, -1, d)[:, :n].double()
        qs = q[i, :heads * d].double().view(kv_heads, group, d)
        p = torch.softmax(qs @ keys.transpose(1, 2) * scale, -1)
        ref[i] = (p @ vals).reshape(heads, d).cpu()
        spread[i] = (p @ vals.abs()).reshape(heads, d).cpu()
    # each probability is rounded to bf16 (half a step, 2^-8 of it at most) on its way to the values, the
    # result once more; scores, exponentials (2 ulp) and sums in fp32 add less than 2^-12 of the spread
    bound = 2.0 ** -8 * (spread + ref.abs()) + 2.0 ** -12 * spread + 1e-30
    return out.view(b, heads, d).double().cpu(), ref, bound


@pytest.mark.gpu
@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("heads, kv_heads, d", [(12, 2, 128), (8, 4, 64), (16, 1, 128), (3, 3, 64), (28, 4, 128)])
def test_against_float64(name, heads, kv_heads, d):
    for slots in (None, 6):
        out, ref, bound = run(CASES[name], heads, kv_heads, d, slots=slots)
        assert ((out - ref).abs() <= bound).all(), ((out - ref).abs() / bound).max()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 3, 5, 10, 11, 21, 22, 33, 64])
def test_rows_of_a_unit(rows):
    for heads, kv_heads in ((6, 1), (2, 2), (15, 1)):
        out, ref, bound = run([(320, [(0, 1 + 7 * i) for i in range(rows)])], heads, kv_heads, 64, seed=rows)
        assert ((out - ref).abs() <= bound).all()


@pytest.mark.gpu
def test_lengths_that_grew_since_the_plan_and_wide_rows():
    prompts = [(300, [(0, 5), (0, 90), (64, 190)])]
    out, ref, bound = run(prompts, 12, 2, 128, plan_at=310, q_pad=512)
    assert ((out - ref).abs() <= bound).all()


@pytest.mark.gpu
def test_a_long_cache():
    out, ref, bound = run([(20000, [(0, 3), (0, 300), (0, 64), (1000, 17)])], 4, 2, 128, poison=False)
    assert ((out - ref).abs() <= bound).all()


@pytest.mark.gpu
def test_scores_that_are_not_finite_stay_in_their_sequence():
    """A NaN or an infinity in what a sequence may see makes its own output NaN and no other's."""
    prompts = [(128, [(0, 9), (0, 70), (0, 1)])]
    tables, lengths, blocks = lists_of(prompts)
    k = torch.randn(blocks, 1, BLOCK, 64, device="cuda").to(torch.bfloat16)
    v = torch.randn(blocks, 1, BLOCK, 64, device="cuda").to(torch.bfloat16)
    k[int(tables[1, 2])] = math.nan                # the second sequence's own block
    v[int(tables[2, 2]), :, 0] = math.inf          # the third one's newest value
    q = torch.randn(3, 2 * 64, device="cuda").to(torch.bfloat16)
    plan = ops.plan_shared(tables, lengths, 2, 1, device="cuda")
    out = ops.shared_decode_attention(q, k, v, torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                                      torch.tensor(tables, dtype=torch.int32, device="cuda"), plan, 2, 1, 64, 0.125)
    assert torch.isfinite(out[0]).all() and out[1].isnan().all() and not torch.isfinite(out[2]).any()


@pytest.mark.gpu
def test_equal_queries_get_equal_bits_and_captured_calls_repeat():
    """Two sequences with the same blocks and the same query have the same output to the bit, call after
    call, eagerly and from a graph (no sum's order depends on chance); the graph reads lengths afresh."""
    heads, kv_heads, d = 12, 2, 128
    tables, lengths, blocks = lists_of([(1000, [(0, 30)] * 6)])
    k = torch.randn(blocks, kv_heads, BLOCK, d, device="cuda").to(torch.bfloat16)
    v = torch.randn_like(k)
    for c in range(tables.shape[0]):                 # (their own last blocks hold the same too)
        k[tables[c, 15:17]], v[tables[c, 15:17]] = k[tables[0, 15:17]], v[tables[0, 15:17]]
    q = torch.randn(1, heads * d, device="cuda").to(torch.bfloat16).repeat(6, 1)
    plan = ops.plan_shared(tables, lengths, heads, kv_heads, device="cuda")
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    table = torch.tensor(tables, dtype=torch.int32, device="cuda")
    call = lambda: ops.shared_decode_attention(q, k, v, lens, table, plan, heads, kv_heads, d, d ** -0.5)
    first = call()
    assert all(torch.equal(first[0], row) for row in first)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = call()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    graph.replay()
    assert torch.equal(first, again) and torch.equal(first, held)
    lens[2] = 1001                                    # (the plan serves shorter tails too)
    graph.replay()
    ops_out = call()
    assert torch.equal(held, ops_out) and torch.equal(held[1], first[1]) and not torch.equal(held[2], first[2])


@pytest.mark.gpu
def test_lengths_that_the_kernel_before_has_written():
    """A call right behind a kernel that lets its successor start early and then writes the lengths reads them as that
    one leaves them."""
    heads, kv_heads, d = 12, 2, 128
    tables, lengths, blocks = lists_of([(1000, [(0, 30), (0, 200), (0, 131)])])
    k = torch.randn(blocks, kv_heads, BLOCK, d, device="cuda").to(torch.bfloat16)
    v = torch.randn_like(k)
    q = torch.randn(3, heads * d, device="cuda").to(torch.bfloat16)
    plan = ops.plan_shared(tables, lengths, heads, kv_heads, device="cuda")
    table = torch.tensor(tables, dtype=torch.int32, device="cuda")
    call = lambda lens: ops.shared_decode_attention(q, k, v, lens, table, plan, heads, kv_heads, d, d ** -0.5)
    want = {}
    for n in (0, 25):
        want[n] = call(torch.tensor(lengths - n, dtype=torch.int32, device="cuda"))
    assert not torch.equal(want[0], want[25])
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    graphs = {}
    for n in want:                  # (captured, so that no time passes between the two; the largest score names the length)
        scores = torch.zeros(3, 2000000, device="cuda")
        scores[range(3), (lengths - n).tolist()] = 1.0
        ops.choose(scores, out=lens), call(lens)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.choose(scores, out=lens)
            out = call(lens)
        graphs[n] = graph, out, scores
    for i in range(20):
        graph, out, _ = graphs[25 * (i % 2)]
        graph.replay()
        assert torch.equal(out, want[25 * (i % 2)])


def test_a_plan_says_which_lengths_it_is_right_for():
    tables, lengths, _ = lists_of(CASES["tree"] + CASES["empty"])
    reach = np.minimum(lengths + 70, tables.shape[1] * BLOCK)
    plan = ops.plan_shared(tables, lengths, 4, 2, slots=20, reach=reach)
    spans = plan.words[plan.span_at:plan.span_at + 2 * len(lengths)].reshape(-1, 2)
    assert (spans[:, 1] == -(-reach // BLOCK) * BLOCK).all()
    for b, row in enumerate(tables):         # the last filled block that another list has in the same place
        shared = [c + 1 for c in range(lengths[b] // BLOCK)
                  if any(o != b and lengths[o] // BLOCK > c and tables[o, c] == row[c] for o in range(len(tables)))]
        assert spans[b, 0] == BLOCK * max(shared, default=0) <= lengths[b]
    assert plan.span_at + 2 * len(lengths) <= len(plan.words)


@pytest.mark.gpu
@pytest.mark.parametrize("heads, kv_heads, d", [(12, 2, 128), (8, 8, 64)])
@pytest.mark.parametrize("forks", [4, 30])
def test_lengths_that_the_plan_does_not_cover(heads, kv_heads, d, forks):
    """No part of an answer: NaN, in the sequence itself and where another's list is read for it; zeros for a
    sequence of no length; all others as they were."""
    tables, lengths, blocks = lists_of([(640, [(0, 30 + i) for i in range(forks)]), (0, [(0, 100)])])
    k = torch.randn(blocks, kv_heads, BLOCK, d, device="cuda").to(torch.bfloat16)
    v = torch.randn_like(k)
    b = len(lengths)
    q = torch.randn(b, heads * d, device="cuda").to(torch.bfloat16)
    plan = ops.plan_shared(tables, lengths, heads, kv_heads, device="cuda", slots=12)
    table = torch.tensor(tables, dtype=torch.int32, device="cuda")

    def call(changed):
        n = lengths.copy()
        for i, to in changed.items():
            n[i] = to
        return ops.shared_decode_attention(q, k, v, torch.tensor(n, dtype=torch.int32, device="cuda"), table, plan,
                                           heads, kv_heads, d, d ** -0.5)

    want = call({})
    assert torch.isfinite(want).all()
    last, alone = forks - 1, forks               # one whose list is read for nobody else, and one that shares nothing
    for length, nan in ((704, False), (640, False), (639, True), (1, True), (705, True), (tables.shape[1] * BLOCK, True),
                        (10 ** 9, True)):
        out = call({last: length})
        assert out[last].isnan().all() if nan else torch.isfinite(out[last]).all()
        rest = [i for i in range(b) if i != last]
        assert torch.equal(out[rest], want[rest])
    for length, nan in ((1, False), (128, False), (129, True)):
        out = call({alone: length})
        assert out[alone].isnan().all() if nan else torch.isfinite(out[alone]).all()
        assert torch.equal(out[:alone], want[:alone])
    for length in (0, -5):
        out = call({last: length, alone: length})
        assert not out[last].any() and not out[alone].any() and torch.equal(out[:last], want[:last])
    first = call({0: 0})                         # the list that is read for all
    assert not first[0].any() and first[1:alone].isnan().all() and torch.equal(first[alone], want[alone])


def test_refusals_of_scales_and_of_plans_that_are_not_there():
    tables, lengths, _ = lists_of(CASES["forks"])
    host = ops.plan_shared(tables, lengths, 12, 2, slots=8)
    plan = host.on(torch.from_numpy(host.words))
    for words in (host.words[:-8], host.words.astype(np.int64), np.repeat(host.words, 2)[::2], host.words[None],
                  np.concatenate([[0], host.words]).astype(np.int32)[1:]):
        with pytest.raises(KernelError, match="words must be"):
            host.on(torch.from_numpy(words))
    b, width = tables.shape
    good = dict(qkv=torch.zeros(b, 12 * 64, dtype=torch.bfloat16), k_cache=torch.zeros(99, 2, 64, 64, dtype=torch.bfloat16),
                v_cache=torch.zeros(99, 2, 64, 64, dtype=torch.bfloat16),
                seq_lens=torch.zeros(b, dtype=torch.int32), block_table=torch.zeros(b, width, dtype=torch.int32),
                plan=plan, heads=12, kv_heads=2, head_dim=64, scale=1.0)
    for scale in (0.0, -0.5, math.nan, math.inf, 1e39, 1e-60):
        with pytest.raises(KernelError, match="scale must be"):
            ops.shared_decode_attention(**{**good, "scale": scale})
    with pytest.raises(KernelError, match="on the host"):
        ops.shared_decode_attention(**{**good, "plan": host})
    for kv_heads in (0, -2):
        with pytest.raises(KernelError):
            ops.shared_decode_attention(**{**good, "kv_heads": kv_heads})
    with pytest.raises(KernelError, match="CUDA device only"):
        ops.shared_decode_attention(**good)


def test_a_plan_of_lists_without_columns():
    plan = ops.plan_shared(np.zeros((3, 0), int), [0, 0, 0], 4, 2, slots=8, roomy=True)
    assert plan.units == plan.unit_capacity == 0 and plan.width == 0


@pytest.mark.gpu
def test_lists_without_columns():
    plan = ops.plan_shared(np.zeros((3, 0), int), [0, 0, 0], 4, 2, device="cuda")
    k = torch.full((2, 2, BLOCK, 64), math.nan, device="cuda", dtype=torch.bfloat16)
    out = ops.shared_decode_attention(torch.ones(3, 256, device="cuda", dtype=torch.bfloat16), k, k,
                                      torch.zeros(3, dtype=torch.int32, device="cuda"),
                                      torch.zeros(3, 0, dtype=torch.int32, device="cuda"), plan, 4, 2, 64, 0.125)
    assert out.shape == (3, 256) and not out.any()


@pytest.mark.gpu
def test_calls_on_two_streams_and_graphs_at_once():
    """Calls side by side, and two captured calls replayed side by side, share nothing."""
    sides = []
    for heads, kv_heads, d, forks in ((12, 2, 128, 9), (8, 4, 64, 40)):
        tables, lengths, blocks = lists_of([(3000, [(0, 5 + 11 * i) for i in range(forks)])])
        k = torch.randn(blocks, kv_heads, BLOCK, d, device="cuda").to(torch.bfloat16)
        v = torch.randn_like(k)
        q = torch.randn(forks, heads * d, device="cuda").to(torch.bfloat16)
        plan = ops.plan_shared(tables, lengths, heads, kv_heads, device="cuda")
        args = (q, k, v, torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                torch.tensor(tables, dtype=torch.int32, device="cuda"), plan, heads, kv_heads, d, d ** -0.5)
        sides.append((args, torch.cuda.Stream()))
    alone = [ops.shared_decode_attention(*args) for args, _ in sides]
    torch.cuda.synchronize()
    got = [[], []]
    for turn in range(10):
        for i, (args, stream) in enumerate(sides):
            with torch.cuda.stream(stream):
                got[i].append(ops.shared_decode_attention(*args, settled=turn % 2 == 1))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, many in zip(alone, got) for b in many)
    graphs = []
    for args, _ in sides:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = [ops.shared_decode_attention(*args, settled=s) for s in (False, True, True)]
        graphs.append((graph, held))
    for args, _ in sides:
        args[0].copy_(args[0].flip(0))
    fresh = [ops.shared_decode_attention(*args) for args, _ in sides]
    torch.cuda.synchronize()
    for _ in range(5):
        for (graph, _), (_, stream) in zip(graphs, sides):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(h, want) for (_, held), want in zip(graphs, fresh) for h in held)
    assert not torch.equal(fresh[0], alone[0])


def test_a_plan_that_no_call_takes_is_refused():
    tables, lengths, _ = lists_of(CASES["forks"])
    assert ops.plan_shared(tables, lengths, 16, 1, slots=8).units
    for heads, kv_heads in ((17, 1), (48, 2), (64, 1)):
        with pytest.raises(KernelError, match="at most 16"):
            ops.plan_shared(tables, lengths, heads, kv_heads, slots=8)

"""Several continuations of one prompt: samples, forks, scores and caches of another size, through the
engine."""

import json

import numpy as np
import pytest
import torch

from semantic_aware_adaptive_kv_cache_precision_b200 import Engine, write_random_model
from semantic_aware_adaptive_kv_cache_precision_b200 import ops
from semantic_aware_adaptive_kv_cache_precision_b200.cache import BLOCK, CacheFull
from semantic_aware_adaptive_kv_cache_precision_b200.engine.generate import plan_samples

from conftest import TINY, prompts_for


def test_plans_of_samples():
    assert plan_samples([100, 64, 1000], 5, 10, 64, 1 << 20) == [[(0, 0, 5), (1, 0, 5), (2, 0, 5)]]
    assert plan_samples([100, 64], 3, 10, 4, 1 << 20) == [[(0, 0, 3), (1, 0, 1)], [(1, 1, 2)]]
    # fifteen whole blocks shared, one of its own each: three fit eighteen blocks
    assert plan_samples([1000], 5, 10, 64, 18 * BLOCK) == [[(0, 0, 3)], [(0, 3, 2)]]
    assert plan_samples([64], 3, 1, 2, 64) == [[(0, 0, 2)], [(0, 2, 1)]]
    with pytest.raises(ValueError, match="request 1 needs"):
        plan_samples([5, 500], 2, 8, 64, 256)
    with pytest.raises(ValueError):
        plan_samples([5], 2, 8, 0, 256)
    rng = np.random.default_rng(0)
    for _ in range(200):
        lens = rng.integers(1, 400, rng.integers(1, 6)).tolist()
        n, new, most = int(rng.integers(1, 9)), int(rng.integers(1, 200)), int(rng.integers(1, 9))
        budget = int(rng.integers(10, 40))
        plan = plan_samples(lens, n, new, most, budget * BLOCK)
        assert [(i, s) for batch in plan for i, a, c in batch for s in range(a, a + c)] == \
            [(i, s) for i in range(len(lens)) for s in range(n)]
        for batch in plan:
            assert sum(c for _, _, c in batch) <= most
            assert sum(lens[i] // BLOCK + c * (-(-(lens[i] + new - 1) // BLOCK) - lens[i] // BLOCK)
                       for i, _, c in batch) <= budget


pytest_gpu = pytest.mark.gpu


def engine_of(folder, dtype="float32", max_tokens=4096, **how):
    return Engine(folder, dtype=dtype, max_tokens=max_tokens, device="cuda:0", **how).load_weights()


@pytest_gpu
@pytest.mark.parametrize("name", ["A", "W", "D"])
@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_samples_are_what_prompts_named_several_times_give(varied_folders, name, temperature):
    """In 32 bits to the last token: a sequence's numbers do not depend on what it shares."""
    engine = engine_of(varied_folders(name), poison_freed=True)
    prompts = prompts_for(name, (70, 5, 64))
    how = dict(temperature=temperature, seed=3, stop_at_eos=False)
    want = engine.generate([p for p in prompts for _ in range(4)], 12, **how)
    seen = []
    got = engine.generate(prompts, 12, samples=4, report=lambda *a: seen.append(a), **how)
    engine.cache.check()
    assert engine.cache.slots.held == 0 and not engine.cache.shares_blocks
    flat = [t for of in got for t in of]
    assert len(got) == 3 and all(len(of) == 4 for of in got)
    assert all(np.array_equal(a, b) for a, b in zip(flat, want))
    assert [e.tokens.tolist() for e in engine.endings] == [t.tolist() for t in flat] and engine.ending is None
    assert {a[3] for a in seen} == set(range(12))
    one = engine.generate(prompts[0], 12, samples=4, **how)
    assert all(np.array_equal(a, b) for a, b in zip(one, want[:4]))
    if temperature:
        assert len({tuple(t) for t in one}) > 1
    assert engine.generate(prompts[1], 0, samples=2, **how)[1].shape == (0,)
    with pytest.raises(ValueError):
        engine.generate(prompts[0], 3, samples=0)


def designs():
    from felovik_configs import CONFIGS as felovik
    from gesuvik_configs import CONFIGS as gesuvik
    from gozolix_configs import CONFIGS as gozolix
    from tebonex_configs import CONFIGS as tebonex
    from venanex_configs import CONFIGS as venanex
    from zodirax_configs import CONFIGS as zodirax
    return {"Tebonex": tebonex["plain"], "Venanex": venanex["mixed"], "Zodirax": zodirax["mixed"],
            "Gesuvik": gesuvik["mixed"], "Felovik": felovik["mixed"], "Gozolix": gozolix["mixed"]}


@pytest_gpu
@pytest.mark.parametrize("design", ["Tebonex", "Venanex", "Zodirax", "Gesuvik", "Felovik", "Gozolix"])
def test_every_design_forks(tmp_path, design):
    """States, latents, windows and tables of pairs go with a fork: in 32 bits samples are to the last token
    what the prompt named several times gives, and scores are the logits' own."""
    config, seed = designs()[design]
    engine = engine_of(write_random_model(tmp_path / design, dict(config), seed, dtype="float32"), poison_freed=True)
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, engine.vocab_size, n) for n in (67, 9)]
    how = dict(temperature=1.0, seed=7, stop_at_eos=False)
    want = engine.generate([p for p in prompts for _ in range(3)], 8, **how)
    got = engine.generate(prompts, 8, samples=3, **how)
    engine.cache.check()
    assert all(np.array_equal(a, b) for a, b in zip([t for of in got for t in of], want))
    check_scores(engine, prompts[0].tolist(), [t.tolist() for t in got[0]] + [[], [3]])


def check_scores(engine, prompt, continuations):
    def plain(ids):
        z = torch.from_numpy(engine.forward(ids)).double()
        return torch.log_softmax(z, -1).numpy()

    # (fp32 logits and sums: a few hundred steps of 2^-24 of the logits' size)
    whole = engine.score(prompt)
    p = plain(prompt)
    np.testing.assert_allclose(whole, p[np.arange(len(prompt) - 1), prompt[1:]], rtol=0, atol=2e-4)
    scores = engine.score(prompt, continuations)
    for c, s in zip(continuations, scores):
        assert s.shape == (len(c),) and s.dtype == np.float32
        p = plain(prompt + c)
        at = np.arange(len(prompt) - 1, len(prompt) + len(c) - 1)
        np.testing.assert_allclose(s, p[at, c], rtol=0, atol=2e-4)
    engine.cache.check()
    assert engine.cache.slots.held == 0


@pytest_gpu
@pytest.mark.parametrize("name", ["A", "B", "W"])
def test_scores_are_the_logits_own(varied_folders, name):
    engine = engine_of(varied_folders(name), max_step_tokens=50)
    vocab = engine.vocab_size
    rng = np.random.default_rng(2)
    prompt = rng.integers(0, vocab, 61).tolist()
    check_scores(engine, prompt, [rng.integers(0, vocab, n).tolist() for n in (1, 2, 7, 40, 0, 1)])
    assert engine.score(prompt[:1]).shape == (0,) and engine.score(prompt, []) == []
    one = engine.score(prompt[:1], [prompt[1:]])[0]
    np.testing.assert_allclose(one, engine.score(prompt), rtol=0, atol=2e-5)
    for bad in (lambda: engine.score([]), lambda: engine.score(prompt, [[vocab]]), lambda: engine.score(prompt, [[1.5]]),
                lambda: engine.score([0] * (engine.spec.max_positions + 1)),
                lambda: engine.score(prompt, [[0] * engine.spec.max_positions])):
        with pytest.raises(ValueError):
            bad()
    assert engine.cache.slots.held == 0


@pytest_gpu
def test_scores_where_the_cache_takes_few_continuations(varied_folders):
    engine = engine_of(varied_folders("A"), max_tokens=4 * BLOCK, max_batch=3)
    rng = np.random.default_rng(3)
    prompt = rng.integers(0, 512, 70).tolist()                  # two blocks; two are left for the forks
    continuations = [rng.integers(0, 512, n).tolist() for n in (20, 30, 40, 5, 50)]
    got = engine.score(prompt, continuations)
    roomy = engine_of(varied_folders("A")).score(prompt, continuations)
    assert all(np.array_equal(a, b) for a, b in zip(got, roomy))
    engine.resize_cache(2 * BLOCK)
    with pytest.raises(CacheFull):
        engine.score(prompt, [[1, 2]])                          # the fork's last block has no room
    engine.cache.check()
    assert engine.cache.slots.held == 0


@pytest_gpu
@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("name", ["D", "C"])
def test_sixteen_bit_steps_over_shared_blocks(varied_folders, name, graphs):
    """Forked sequences step like sequences of their own, within what bfloat16 leaves of a logit, and the
    choice of tokens inside the captured step follows its own logits."""
    engine = engine_of(varied_folders(name, "bfloat16"), "bfloat16", cuda_graphs=graphs, max_tokens=8192)
    alone = engine_of(varied_folders(name, "bfloat16"), "bfloat16", cuda_graphs=graphs, max_tokens=8192)
    engine.shared_bytes_worth, alone.shared_bytes_worth = 0, None
    assert (len(engine.model.shared_readers()) > 0) == (name in "DC")
    rng = np.random.default_rng(4)
    vocab, prompt = engine.vocab_size, rng.integers(0, engine.vocab_size, 450).tolist()
    steps = rng.integers(0, vocab, (75, 7))
    out = []
    for e in (engine, alone):
        (a,) = e.open(1)
        e.step([a], [prompt])
        slots = [a] + e.fork(a, 4)
        rows = []
        for i, tokens in enumerate(steps):
            if i == 20:                       # a fork of a fork, and one leaves
                slots = slots + e.fork(slots[2], 2)
            if i == 40:
                e.close([slots.pop(1)])
            rows.append(e.step(slots, [[int(t)] for t in tokens[:len(slots)]]).cpu())
            if e is engine:
                assert e.cache.shares_blocks and e._shared_now[2]
        greedy = e.next_tokens(slots, torch.zeros(len(slots), dtype=torch.int32, device="cuda")).cpu()
        out.append((rows, greedy, slots))
        e.close(slots)
        e.cache.check()
    assert alone._shared_now is None
    for a, b in zip(out[0][0], out[1][0]):
        assert a.shape == b.shape
        assert ((a - b).abs() <= 0.06 * b.std(-1, keepdim=True)).all()


@pytest_gpu
def test_a_captured_step_reads_the_plan_of_the_moment(varied_folders):
    """The same batch shape with other sequences sharing: graphs are shared between plans of one layout, and
    every one reads its own."""
    engine = engine_of(varied_folders("D", "bfloat16"), "bfloat16", max_tokens=16384)
    engine.shared_bytes_worth = 0
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, 400, 200).tolist() for _ in range(2)]
    heads = engine.open(2)
    engine.step(heads, prompts)
    first = [heads[0]] + engine.fork(heads[0], 3)
    second = [heads[1]] + engine.fork(heads[1], 3)
    mixed = [first[1], second[1], second[2], first[2]]
    want = {}
    for round in range(3):
        for group in (first, second, mixed, first[::-1]):
            logits = engine.step(group, [[7]] * 4).cpu()
            for s, row in zip(group, logits):
                n = int(engine.cache.lengths[s])
                key = (s in first, n)
                if key in want:      # (the same tokens behind the same prompt, in whatever company)
                    assert ((row - want[key]).abs() <= 0.06 * row.std()).all()
                want.setdefault(key, row)
    engine.close(first + second)
    engine.cache.check()


@pytest_gpu
def test_captured_steps_that_want_some_logits_ask_whether_blocks_are_shared(varied_folders):
    """A step of one token a sequence that does not want every logit is captured by its counts and starts: with
    the same ones and nothing shared it is another step."""
    engine = engine_of(varied_folders("D", "bfloat16"), "bfloat16", max_tokens=8192)
    engine.shared_bytes_worth = 0
    rng = np.random.default_rng(8)
    prompts = [rng.integers(0, 400, 200).tolist() for _ in range(3)]

    def wanted(slots):
        out = engine.step(slots, [[5], [6], [7]], [[0], [], [0]]).cpu()
        engine.close(slots)
        return out

    def shared(prompt):
        (a,) = engine.open(1)
        engine.step([a], [prompt])
        return [a] + engine.fork(a, 2)

    def alone(prompt):
        slots = engine.open(3)
        engine.step(slots, [prompt] * 3)
        return slots

    for prompt in prompts:                  # (the second time the shape comes up it is captured, the third replayed)
        a, b = wanted(shared(prompt)), wanted(alone(prompt))
        assert ((a - b).abs() <= 0.06 * b.std(-1, keepdim=True)).all()


@pytest_gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_cache_of_another_size_between_steps(varied_folders, dtype):
    engine = engine_of(varied_folders("A", dtype), dtype, max_tokens=1024)
    same = engine_of(varied_folders("A", dtype), dtype, max_tokens=1024)
    rng = np.random.default_rng(6)
    prompt = rng.integers(0, 512, 40).tolist()
    outs = []
    for e in (engine, same):
        gone, a = e.open(2)
        e.step([gone, a], [prompt[:30], prompt])
        slots = [a] + e.fork(a, 2)
        e.close([gone])
        rows = []
        for i in range(30):
            if e is engine and i in (5, 15):
                e.resize_cache(4 * BLOCK if i == 5 else 8192)
                e.cache.check()
            rows.append(e.step(slots, [[i], [2 * i], [3 * i]]).cpu())
        e.close(slots)
        outs.append(torch.stack(rows))
    assert torch.equal(outs[0], outs[1])
    assert engine.max_tokens == 8192 and engine.cache.max_seq_len == 128
    with pytest.raises(ValueError):
        engine.resize_cache(0)
    (a,) = engine.open(1)
    engine.step([a], [prompt * 2])
    with pytest.raises(CacheFull):
        engine.resize_cache(BLOCK)
    assert engine.max_tokens == 8192
    engine.close([a])
    assert all(len(g) == 3 for g in engine.generate([prompt] * 40, 3, stop_at_eos=False))     # slots grew too
    engine.resize_cache(BLOCK)
    assert engine.generate(prompt, 5, stop_at_eos=False).shape == (5,)


@pytest_gpu
def test_samples_that_end_and_a_full_cache(varied_folders):
    engine = engine_of(varied_folders("D", "bfloat16"), "bfloat16", max_tokens=40 * BLOCK)
    engine.shared_bytes_worth = 0
    prompt = prompts_for("D", (300,))[0]
    free = engine.generate(prompt, 30, samples=12, temperature=1.0, seed=1, stop_at_eos=False)
    stops = {int(free[0][4]), int(free[5][9])}
    got = engine.generate(prompt, 30, samples=12, temperature=1.0, seed=1, stop_token_ids=stops)
    engine.cache.check()
    assert engine.cache.slots.held == 0 and any(len(g) < 30 for g in got)
    for g, e in zip(got, engine.endings):
        assert e.reason == ("stop" if int(g[-1]) in stops else "length")
        assert not any(int(t) in stops for t in g[:-1])
    held = engine.open(3)                                    # another user's sequences leave too little
    engine.step(held, [prompt.tolist() * 2] * 3)
    full = engine.generate(prompt, 30, samples=12, temperature=1.0, seed=1, stop_at_eos=False)
    assert len(full) == 12 and all(e.state == "exhausted" for e in engine.endings)
    engine.cache.check()
    assert engine.cache.slots.held == 3
    engine.close(held)


@pytest_gpu
def test_targets_of_a_step(varied_folders):
    engine = engine_of(varied_folders("A"))
    a, b = engine.open(2)
    got = engine.step([a, b], [[1, 2, 3], [4, 5]], [[0, 2, 2], []], targets=[[7, 8, 511], []])
    assert got.shape == (3,) and got.dtype == torch.float32
    z = torch.log_softmax(torch.from_numpy(engine.forward([1, 2, 3])).double(), -1)
    np.testing.assert_allclose(got.cpu().numpy(), [z[0, 7], z[2, 8], z[2, 511]], rtol=0, atol=2e-4)
    assert engine.step([a, b], [[1], [2]], [[], []], targets=[[], []]).shape == (0,)
    lengths = engine.cache.lengths[[a, b]].tolist()
    for how in (dict(targets=[[1, 2], [3]]), dict(targets=[[1]]), dict(targets=[[512], [3]]), dict(targets=[[-1], [3]]),
                dict(targets=[[1], [3]], hidden_states=[])):
        with pytest.raises(ValueError):
            engine.step([a, b], [[1], [2]], **how)
    assert engine.cache.lengths[[a, b]].tolist() == lengths
    engine.close([a, b])


@pytest_gpu
def test_little_that_is_shared_is_read_by_everyone(varied_folders):
    """Below the bytes that pay, no plan is made and the step is the one of sequences of their own, to the bit."""
    engine = engine_of(varied_folders("D", "bfloat16"), "bfloat16")
    rng = np.random.default_rng(9)
    prompt = rng.integers(0, 400, 300).tolist()
    (a,) = engine.open(1)
    engine.step([a], [prompt])
    slots = [a] + engine.fork(a, 3)
    out = [engine.step(slots, [[t]] * 4).cpu() for t in (1, 2, 3)]
    assert engine._shared_now[2] == {} and not engine._shared_buffers
    assert all(torch.equal(o[0], row) for o in out for row in o)
    engine.close(slots)
    engine.shared_bytes_worth = None
    (a,) = engine.open(1)
    engine.step([a], [prompt])
    slots = [a] + engine.fork(a, 3)
    assert all(torch.equal(o, engine.step(slots, [[t]] * 4).cpu()) for o, t in zip(out, (1, 2, 3)))
    engine.close(slots)


@pytest_gpu
def test_the_command_line(varied_folders, capsys):
    from semantic_aware_adaptive_kv_cache_precision_b200.cli import main
    folder = str(varied_folders("A"))
    assert main(["generate", "--model", folder, "--dtype", "float32", "--prompt-ids", "1,2,3", "--prompt-ids", "4",
                 "--new-tokens", "5", "--samples", "3", "--temperature", "1.0", "--ignore-eos"]) == 0
    lines = [json.loads(x) for x in capsys.readouterr().out.splitlines()]
    assert [x["request"] for x in lines] == list(range(6)) and all(len(x["tokens"]) == 5 for x in lines)
    assert main(["score", "--model", folder, "--dtype", "float32", "--prompt-ids", "1,2,3",
                 "--continuation-ids", "4,5", "--continuation-ids", "6"]) == 0
    lines = [json.loads(x) for x in capsys.readouterr().out.splitlines()]
    assert [x["tokens"] for x in lines] == [2, 1] and abs(sum(lines[0]["logprobs"]) - lines[0]["logprob"]) < 1e-5
    assert main(["score", "--model", folder, "--dtype", "float32", "--prompt-ids", "1,2,3"]) == 0
    line = json.loads(capsys.readouterr().out)
    assert line["prompt"] == 0 and line["tokens"] == 2


def engine_without_a_gpu(monkeypatch, cache, readers):
    """An engine's bookkeeping of plans over a cache on the host, with nothing that launches."""
    from types import SimpleNamespace
    from semantic_aware_adaptive_kv_cache_precision_b200.engine import engine as module
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda t: t)
    monkeypatch.setattr(module._lib, "sm_count", lambda device=None: 148)
    e = Engine.__new__(Engine)
    e.device, e.cache, e.model = torch.device("cpu"), None, SimpleNamespace(shared_readers=lambda: readers, arena=None)
    e.shared_bytes_worth, e._shared_now, e._shared_buffers, e._shared_readers = 0, None, {}, None
    e._shared_known = {}
    e._graphs, e._prefill_graphs = {}, {}
    return e


def test_captured_steps_go_with_the_plans_they_read(monkeypatch):
    """A captured step reads its plan at a device address. When the buffers of plans are given up, every captured
    step whose key has a plan is, however it was captured: the next plan of that layout lies elsewhere."""
    from types import SimpleNamespace
    from semantic_aware_adaptive_kv_cache_precision_b200.cache import KVNeed, SequenceCache
    from semantic_aware_adaptive_kv_cache_precision_b200.engine import engine as module
    monkeypatch.setattr(module, "MOST_PLAN_BUFFERS", 3, raising=False)
    need = KVNeed(1, 64)
    cache = SequenceCache([need], 64 * BLOCK, 64 * BLOCK, torch.bfloat16, "cpu", max_slots=90)
    e = engine_without_a_gpu(monkeypatch, cache, [(need, 2)])
    (a,) = cache.open(1)
    cache.reserve([a], [2 * BLOCK])
    cache.advance([a], [2 * BLOCK])
    slots = [a] + cache.fork(a, 80)
    for n in list(range(2, 75)) + [2, 40]:
        plans = e._shared_plans(slots[:n], [2 * BLOCK] * n, cache)
        assert plans
        key = ("step", n, module._plans_in_key(SimpleNamespace(shared=plans)))
        at = [plan.words.data_ptr() for plan in plans.values()]
        for table in (e._graphs, e._prefill_graphs):
            if key in table:           # (it would be replayed)
                assert table[key] == at
            table[key] = at
        assert len(e._shared_buffers) <= 64
        held = {b.data_ptr() for b, _ in e._shared_buffers.values()}
        assert all(set(x) <= held for table in (e._graphs, e._prefill_graphs) for x in table.values())


def test_a_size_whose_tables_find_no_room_changes_nothing(monkeypatch):
    """The tables of positions are made before the cache changes, and never for fewer positions than it takes."""
    import contextlib
    from semantic_aware_adaptive_kv_cache_precision_b200.cache import KVNeed, SequenceCache
    from semantic_aware_adaptive_kv_cache_precision_b200.errors import OutOfDeviceMemory
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    cache = SequenceCache([KVNeed(1, 64)], 8 * BLOCK, 64 * BLOCK, torch.bfloat16, "cpu")
    e = engine_without_a_gpu(monkeypatch, cache, [])
    e.cache, e.max_tokens, asked = cache, 8 * BLOCK, []

    def prepare(n):
        asked.append(n)
        if n > 30 * BLOCK:
            raise torch.OutOfMemoryError("no room")

    e.model.prepare = prepare
    (a,) = cache.open(1)
    cache.reserve([a], [100])
    cache.advance([a], [100])
    keys, table = cache.groups[0].keys, cache.groups[0].tables.copy()
    e._graphs["step"] = e._prefill_graphs["step"] = object()
    with pytest.raises(OutOfDeviceMemory):
        e.resize_cache(40 * BLOCK)
    cache.check()
    assert cache.max_seq_len == e.max_tokens == 8 * BLOCK and cache.groups[0].keys is keys
    assert (cache.groups[0].tables == table).all()
    assert not e._graphs and not e._prefill_graphs         # (tables of some layers may be new ones)
    e._graphs["step"] = object()
    with pytest.raises(CacheFull):
        e.resize_cache(BLOCK)                              # refused before anything is made or dropped
    assert asked == [40 * BLOCK] and e._graphs and e.max_tokens == 8 * BLOCK
    e.resize_cache(20 * BLOCK)
    assert cache.max_seq_len == e.max_tokens == 20 * BLOCK and not e._graphs
    e.resize_cache(4 * BLOCK)
    assert cache.max_seq_len == 4 * BLOCK and asked[1:] == [20 * BLOCK, 20 * BLOCK]
    cache.check()


def test_rotary_tables_are_made_both_or_neither(monkeypatch):
    from types import SimpleNamespace
    from semantic_aware_adaptive_kv_cache_precision_b200.parts.rotary import RotaryHalf
    part = RotaryHalf(SimpleNamespace(rotary_dim=8, head_dim=8, max_positions=100, theta=1e4, scaling=None), "", None)
    part.prepare("cpu", 10)
    moved, to = [], torch.Tensor.to

    def full(t, *args, **how):
        moved.append(t)
        if len(moved) == 2:
            raise torch.OutOfMemoryError("no room")
        return to(t, *args, **how)

    with monkeypatch.context() as m:
        m.setattr(torch.Tensor, "to", full)
        with pytest.raises(torch.OutOfMemoryError):
            part.prepare("cpu", 50)
    assert part.cos.shape == part.sin.shape == (10, 4)
    part.prepare("cpu", 50)
    assert part.cos.shape == part.sin.shape == (50, 4)


def test_a_window_that_slides_leaves_the_plans_of_other_groups(monkeypatch):
    """Blocks that a window's group gives back are none that a plan speaks of."""
    from semantic_aware_adaptive_kv_cache_precision_b200.cache import KVNeed, SequenceCache
    whole, window = KVNeed(1, 64), KVNeed(2, 64, window=100)
    cache = SequenceCache([whole, window], 40 * BLOCK, 40 * BLOCK, torch.bfloat16, "cpu", max_slots=9)
    e = engine_without_a_gpu(monkeypatch, cache, [(whole, 2)])
    made = []
    plan_shared = ops.plan_shared
    monkeypatch.setattr(ops, "plan_shared", lambda *args, **how: (made.append(args[1]), plan_shared(*args, **how))[1])

    def grow(slots, n):
        cache.reserve(slots, [n] * len(slots))
        plans = e._shared_plans(slots, [n] * len(slots), cache)
        cache.advance(slots, [n] * len(slots))
        return plans

    (a,) = cache.open(1)
    grow([a], 4 * BLOCK)
    slots = [a] + cache.fork(a, 3)
    for n in range(4 * BLOCK + 1, 8 * BLOCK):        # the window leaves every block that the four share behind
        assert grow(slots, n)
    cache.check()
    assert len(made) == 1 and cache.groups[1].sharing > cache.groups[0].sharing
    b = cache.fork(a, 1)
    assert grow(slots + b, 8 * BLOCK) and len(made) == 2
    cache.close(b)
    assert grow(slots, 8 * BLOCK + 1) and len(made) == 3


def counted_plans(monkeypatch):
    made, plan_shared = [], ops.plan_shared
    monkeypatch.setattr(ops, "plan_shared", lambda *args, **how: (made.append(len(args[1])), plan_shared(*args, **how))[1])
    return made


def test_batches_that_step_in_turn_keep_their_plans(monkeypatch):
    """And each reads its own, also where two lie at one address; a batch that shares nothing asks for no plan."""
    from semantic_aware_adaptive_kv_cache_precision_b200.cache import KVNeed, SequenceCache
    from semantic_aware_adaptive_kv_cache_precision_b200.engine import engine as module
    need = KVNeed(1, 64)
    cache = SequenceCache([need], 64 * BLOCK, 64 * BLOCK, torch.bfloat16, "cpu", max_slots=60)
    e = engine_without_a_gpu(monkeypatch, cache, [(need, 2)])
    e.shared_bytes_worth = 4 * 2 * 64 * 64 * 2           # four blocks of keys and values
    made = counted_plans(monkeypatch)
    heads = cache.open(4)
    cache.reserve(heads, [4 * BLOCK, 4 * BLOCK, 3 * BLOCK, 2 * BLOCK])
    cache.advance(heads, [4 * BLOCK, 4 * BLOCK, 3 * BLOCK, 2 * BLOCK])
    first, second = ([h] + cache.fork(h, 3) for h in heads[:2])
    alone = heads[2:]
    mixed = [first[0], second[0], heads[2], heads[3]]    # as many sequences, nothing shared among them
    lists = {}
    for turn in range(20):
        for name, slots in (("first", first), ("second", second), ("mixed", mixed), ("alone", alone)):
            now = [int(cache.lengths[s]) + 1 for s in slots]
            cache.reserve(slots, now)
            plans = e._shared_plans(slots, now, cache)
            assert bool(plans) == (name in ("first", "second"))
            if plans:
                plan = plans[0, 2]
                fresh = ops.plan_shared(cache.tables_for(slots)[0][:, :plan.width], now, 2, 1, None, reach=plan.reach,
                                        roomy=True, slots=296)
                made.pop()
                lists.setdefault(name, plan.words.data_ptr())
                assert lists[name] == plan.words.data_ptr() and np.array_equal(plan.words.numpy(), fresh.words)
    assert lists["first"] == lists["second"]             # (one layout)
    assert made == [4, 4]
    for i in range(20):                                  # batches come and go: no more than some are kept
        slots = first[:2 + i % 3] + alone[:i % 2]
        e._shared_plans(slots, [int(cache.lengths[s]) + 1 for s in slots], cache)
        assert len(e._shared_known) <= module.KNOWN_PLANS
    e.shared_bytes_worth = 10 ** 12                      # what pays is asked anew
    assert e._shared_plans(first, [4 * BLOCK + 2] * 4, cache) == {}
    e.shared_bytes_worth = 0
    assert e._shared_plans(first, [4 * BLOCK + 2] * 4, cache)


@pytest_gpu
@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("worth", [0, None])
def test_chosen_tokens_over_shared_blocks_are_the_logits_best(varied_folders, graphs, worth):
    """`next_tokens` chooses inside the step, captured or not: its tokens have the largest logits that `step` gives equal
    forks that are fed the same, and lead to the same places."""
    engine = engine_of(varied_folders("D", "bfloat16"), "bfloat16", cuda_graphs=graphs, max_tokens=16384)
    engine.shared_bytes_worth = worth
    rng = np.random.default_rng(11)
    (a,) = engine.open(1)
    engine.step([a], [rng.integers(0, engine.vocab_size, 450).tolist()])
    slots = engine.fork(a, 4)
    fed = torch.tensor([3, 77, 150, 399], dtype=torch.int32, device="cuda")
    twins = engine.fork(a, 4)
    seen = set()
    for _ in range(12):
        logits = engine.step(twins, device_tokens=fed.clone())
        if worth == 0:
            assert engine._shared_now[2]
        fed = engine.next_tokens(slots, fed).clone()
        best, mine = logits.amax(1), logits.gather(1, fed.long()[:, None])[:, 0]
        # (both steps are bfloat16 steps of the same sequences: as far apart as such steps are)
        assert ((best - mine) <= 0.06 * logits.std(1)).all()
        seen.update(fed.tolist())
    assert len(seen) > 4
    engine.close([a] + slots + twins)
    engine.cache.check()


@pytest_gpu
@pytest.mark.parametrize("what", ["resize", "many shapes", "many plans"])
def test_steps_are_captured_again_after_all_captured_ones_have_gone(varied_folders, monkeypatch, what):
    """Also where something that lies in their memory is still held, as scratch that a capture made may be."""
    from semantic_aware_adaptive_kv_cache_precision_b200.engine import engine as module
    engine = engine_of(varied_folders("D", "bfloat16"), "bfloat16", max_tokens=16384)
    engine.shared_bytes_worth = 0
    (a,) = engine.open(1)
    engine.step([a], [list(range(200))])
    slots = [a] + engine.fork(a, 4)
    for _ in range(3):
        engine.step(slots, [[7]] * 5)
    assert len(engine._graphs) == 1 and engine._shared_buffers
    held = [entry[1] for entry in engine._graphs.values()]
    if what == "resize":
        engine.resize_cache(20000)
    elif what == "many shapes":
        graph = next(iter(engine._graphs.values()))
        engine._graphs.update({i: graph for i in range(63)})
        del graph
    else:
        monkeypatch.setattr(module, "MOST_PLAN_BUFFERS", 1)
    for n in (4, 5, 4, 5):
        engine.step(slots[:n], [[7]] * n)
    assert engine.cuda_graphs and engine.graph_failure is None and engine._graphs
    assert held[0].shape[0] == 5
    engine.close(slots)
    engine.cache.check()

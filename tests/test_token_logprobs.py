"""Log-probabilities of given tokens without keeping the logits, against float64."""

import math

import pytest
import torch

from semantic_aware_adaptive_kv_cache_precision_b200 import ops
from semantic_aware_adaptive_kv_cache_precision_b200.ops import KernelError, logprobs


def test_refusals():
    x, w, t = torch.zeros(3, 16), torch.zeros(50, 16), torch.zeros(3, dtype=torch.int32)
    call = ops.token_logprobs
    for args, how in (((x, w[:, :8], t), {}), ((x, w.to(torch.bfloat16), t), {}), ((x, w[::2], t), {}),
                      ((x[:, ::2], w[:, :8].contiguous(), t), {}), ((x, w, t.long()), {}), ((x, w, t[:2]), {}),
                      ((x, w, t, torch.zeros(49)), {}), ((x, w, t, torch.zeros(50).double()), {}),
                      ((x, w[:0], t), {}), ((x[:, :0], w[:, :0], t), {}), ((x, w, t), {"softcap": -1.0}),
                      ((x, w, t), {"softcap": math.inf}), ((x, w, t), {"softcap": math.nan}),
                      ((x.double(), w.double(), t), {}), ((x[:1].expand(3, 16), w, t), {}),
                      ((torch.zeros(40).as_strided((3, 16), (4, 1)), w, t), {})):
        with pytest.raises(KernelError):
            call(*args, **how)
    with pytest.raises(KernelError, match="CUDA device only"):
        call(x, w, t)


def reference(x, w, targets, bias, scale, softcap):
    z = x.double() @ w.double().t()
    size = x.double().abs() @ w.double().abs().t()          # of the products whose sum a logit is
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs().nan_to_num(0, 0, 0)
    z, size = z * scale, size * abs(scale)
    if softcap:
        z = softcap * torch.tanh(z / softcap)
    lse = torch.logsumexp(z, 1)
    picked = z.gather(1, targets.long().clamp(0, w.shape[0] - 1)[:, None])[:, 0]
    # a logit is a sum of K products in fp32, every addition off by a step at most (2^-23 of what it adds up:
    # the tensor cores cut off), then the cap's tanh by 2^-21 of the cap; lse moves by no more than the largest
    # of them, and its own sum of V positive terms in runs of at most 512 by 512 2^-23, its logarithm by 2^-21
    k = x.shape[1]
    dz = ((k + 4) * 2.0 ** -23 * size).amax(1) + 2.0 ** -21 * softcap
    return picked - lse, lse, 2 * dz + 512 * 2.0 ** -23 + 2.0 ** -21 * (1 + lse.abs()) + 2.0 ** -22 * picked.abs()


def check(rows, k, vocab, dtype, bias=None, scale=1.0, softcap=0.0, seed=0, x_pad=0, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, k + x_pad), generator=g, device="cuda").to(dtype)[:, :k]
    w = (torch.randn((vocab, k), generator=g, device="cuda") * spread / math.sqrt(k)).to(dtype)
    b = None if bias is None else torch.randn(vocab, generator=g, device="cuda").to(bias)
    targets = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    targets[0], targets[-1] = vocab - 1, 0
    got, lse = ops.token_logprobs(x, w, targets, b, scale=scale, softcap=softcap)
    want, want_lse, bound = reference(x, w, targets, b, scale, softcap)
    assert ((lse.double() - want_lse).abs() <= bound).all(), ((lse.double() - want_lse).abs() / bound).max()
    assert ((got.double() - want).abs() <= bound).all(), ((got.double() - want).abs() / bound).max()
    return x, w, targets, got, lse


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows, k, vocab", [(1, 8, 1), (1, 64, 255), (5, 96, 256), (31, 72, 257), (127, 128, 1000),
                                            (129, 192, 4095), (256, 64, 4097), (257, 200, 8193), (600, 256, 70001), (255, 64, 3000), (333, 136, 20000),
                                            (511, 64, 128), (40, 1024, 40000), (96, 64, 5000), (97, 64, 5000),
                                            (384, 72, 5000), (385, 72, 5000), (608, 64, 5000), (609, 64, 5000)])
def test_against_float64(dtype, rows, k, vocab):
    check(rows, k, vocab, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bias", [None, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale, softcap", [(1.0, 0.0), (0.25, 0.0), (1.0, 5.0), (-0.5, 30.0)])
def test_bias_scale_and_cap(dtype, bias, scale, softcap):
    for rows in (70, 130, 300, 700):
        check(rows, 104, 1333, dtype, bias, scale, softcap)
    check(3, 104, 1333, dtype, bias, scale, softcap, spread=40.0)


@pytest.mark.parametrize("pairs", [1, 7, 74])
def test_tiles_cover_the_vocabulary(pairs):
    """Host code of the launcher: every row of the head in one tile, tiles no higher than a block's rows, and no
    more pairs than tiles. (Needs nvcc, not a GPU.)"""
    import ctypes
    from semantic_aware_adaptive_kv_cache_precision_b200.ops._lib import plain_function
    shape = (ctypes.c_int * 4)()
    for rows in (1, 31, 96, 97, 255, 256, 257, 333, 384, 385, 511, 513, 608, 609, 2047, 2048):
        for vocab, k in ((v, k) for v in (1, 2, 300, 4097, 50257, 151936) for k in (64, 1024, 1032)):
            assert plain_function("sakv_logprob_shape")(rows, vocab, k, pairs, shape) == 0
            full, height, tiles, launched = shape
            rest = rows - 256 * full
            per = 1 if full == 1 and rest > 0 and k <= 1024 else full + (rest > 0)
            assert rest <= (128 if k <= 1024 else 96)
            assert rest > -256 and 1 <= height <= 128 and (not full or height % 16 == 0)
            assert (tiles - 1) * 2 * height < vocab <= tiles * 2 * height
            assert launched == min(pairs, tiles * per)
            if not full:                      # every block has the same number of rows in all, but for the last ones
                assert -(-tiles // launched) * 2 * height * launched - vocab < 2 * launched * -(-tiles // launched)
    for bad in ((0, 5, 64, 1), (5, 0, 64, 1), (5, 5, 0, 1), (5, 5, 64, 0), (2 ** 31 - 1, 5, 64, 1)):
        assert plain_function("sakv_logprob_shape")(*bad, shape) != 0


@pytest.mark.gpu
def test_operands_that_the_copies_do_not_take():
    check(20, 37, 500, torch.bfloat16)                     # rows of the head at odd addresses
    check(20, 37, 500, torch.float32)
    check(33, 64, 500, torch.bfloat16, x_pad=3)            # rows of x likewise
    check(33, 64, 500, torch.bfloat16, x_pad=24)           # rows a multiple of 16 bytes apart
    check(40, 64, 500, torch.float32, x_pad=3)
    for dtype in (torch.bfloat16, torch.float32):
        check(5, 1, 300, dtype)                            # one number a row
        x, w, targets, got, lse = check(1, 64, 300, dtype)
        again, _ = ops.token_logprobs(x.as_strided((1, 64), (0, 1)), w, targets)     # a row's own stride means nothing
        assert torch.equal(again, got)


@pytest.mark.gpu
def test_pieces_of_rows_where_logits_lie_in_memory(monkeypatch):
    x, w, targets, got, lse = check(50, 47, 9000, torch.bfloat16, seed=5)
    monkeypatch.setattr(logprobs, "PIECE_ELEMENTS", 17 * 4096)
    again, lse2 = ops.token_logprobs(x, w, targets)
    # (the library's product of these rows sums in another order when its shape is another)
    want, want_lse, bound = reference(x, w, targets, None, 1.0, 0.0)
    assert ((again.double() - want).abs() <= bound).all() and ((lse2.double() - want_lse).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_targets_that_ask_for_nothing_and_masked_tokens(dtype):
    rows, k, vocab = 9, 64, 700
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((rows, k), generator=g, device="cuda").to(dtype)
    w = torch.randn((vocab, k), generator=g, device="cuda").mul_(0.3).to(dtype)
    bias = torch.zeros(vocab, device="cuda")
    bias[300:] = -math.inf                                   # whole pieces of the vocabulary
    bias[::2] = -math.inf
    targets = torch.tensor([1, 299, 3, 2, 500, -1, -2 ** 31, vocab, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    got, lse = ops.token_logprobs(x, w, targets, bias)
    want, want_lse, bound = reference(x, w, targets, bias, 1.0, 0.0)
    assert ((lse.double() - want_lse).abs() <= bound).all()
    assert ((got.double() - want)[:3].abs() <= bound[:3]).all()
    assert (got[3:5] == -math.inf).all() and (got[5:7] == 0).all() and got[7:].isnan().all()
    lowest = torch.finfo(torch.float32).min                  # a mask of the type's lowest value does the same
    same, lse2 = ops.token_logprobs(x, w, targets, bias.clamp(min=lowest))
    assert torch.equal(lse, lse2) and torch.equal(got[:3], same[:3]) and (same[3:5] < -1e38).all()
    bias[:] = lowest                                         # everything masked so: all tokens alike, in 32 bits 0
    got, lse = ops.token_logprobs(x, w, targets, bias)
    assert (lse <= lowest / 2).all() and torch.isfinite(lse).all() and (got[:5].abs() <= 1e32).all()
    bias[:] = -math.inf
    got, lse = ops.token_logprobs(x, w, targets, bias)
    assert (lse == -math.inf).all() and got[:5].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_rows_that_are_not_finite_stay_their_own(dtype, softcap):
    x = torch.randn(40, 64, device="cuda").to(dtype)
    w = torch.randn(900, 64, device="cuda").mul_(0.3).to(dtype)
    targets = torch.arange(40, dtype=torch.int32, device="cuda")
    good, _ = ops.token_logprobs(x, w, targets, softcap=softcap)
    x[7] = math.nan
    got, lse = ops.token_logprobs(x, w, targets, softcap=softcap)
    assert got[7].isnan() and lse[7].isnan()
    rest = [i for i in range(40) if i != 7]
    assert torch.equal(got[rest], good[rest])


@pytest.mark.gpu
def test_no_rows_rows_alone_streams_and_graphs():
    x, w, targets, got, lse = check(300, 128, 3001, torch.bfloat16, seed=9)
    none, none_lse = ops.token_logprobs(x[:0], w, targets[:0])
    assert none.shape == none_lse.shape == (0,)
    # in 32 bits a row's sums do not depend on the rows beside it
    wide, head = x.float(), w.float()
    whole, _ = ops.token_logprobs(wide, head, targets)
    for n in (7, 16, 30, 64):
        some, _ = ops.token_logprobs(wide[5:5 + n], head, targets[5:5 + n])
        assert torch.equal(some, whole[5:5 + n])
    for i in (0, 130, 299):
        alone, _ = ops.token_logprobs(wide[i:i + 1], head, targets[i:i + 1])
        assert torch.equal(alone, whole[i:i + 1])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again, _ = ops.token_logprobs(x, w, targets)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held, _ = ops.token_logprobs(x, w, targets)
    graph.replay()
    assert torch.equal(again, got) and torch.equal(held, got)
    x.copy_(x.flip(0))
    graph.replay()
    fresh, _ = ops.token_logprobs(x, w, targets)
    assert torch.equal(held, fresh) and not torch.equal(held, got)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [32, 33, 64, 65, 96, 97, 128, 129, 257])
@pytest.mark.parametrize("k, vocab", [(4, 104), (60, 129), (68, 1000), (128, 127), (132, 15500), (260, 20000), (1028, 333)])
def test_numbers_of_32_bits_in_three(rows, k, vocab):
    check(rows, k, vocab, torch.float32, x_pad=(rows + k // 4) % 3, seed=rows + k)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [640, 4096])
def test_long_sums_of_32_bits(k):
    """Numbers of one sign, where what is cut off adds up."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.rand((40, k), generator=g, device="cuda") + 0.5
    w = (torch.rand((700, k), generator=g, device="cuda") + 0.5) / k
    targets = torch.randint(0, 700, (40,), generator=g, device="cuda", dtype=torch.int32)
    got, lse = ops.token_logprobs(x, w, targets)
    z = x.double() @ w.double().t()
    want_lse = torch.logsumexp(z, 1)
    want = z.gather(1, targets.long()[:, None])[:, 0] - want_lse
    # the sums of 128 products are taken off the tensor cores, where each product and each of eight additions is cut
    # by a step of the sum (2^-23) at most; what is left out of a product is 2^-21 of it; the k / 128 additions of
    # those sums round by 2^-24; lse's own sum as above
    dz = (136 + 4 + k / 256) * 2.0 ** -23 * z.amax()
    assert ((lse.double() - want_lse).abs() <= dz + 512 * 2.0 ** -23 + 2.0 ** -21 * (1 + want_lse)).all()
    assert ((got.double() - want).abs() <= 2 * dz + 512 * 2.0 ** -23 + 2.0 ** -21 * (2 + want_lse)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("name, value", [("SPLIT_ELEMENTS", 70 * 136), ("SPLIT_PAIRS", 29 * 101)])
def test_rows_of_32_bits_in_pieces(monkeypatch, name, value):
    x, w, targets, got, lse = check(301, 132, 3001, torch.float32, seed=8)
    monkeypatch.setattr(logprobs, name, value)
    again, lse2 = ops.token_logprobs(x, w, targets)
    assert torch.equal(again, got) and torch.equal(lse, lse2)


def test_heights_and_widths_of_32_bit_tiles():
    """Host code of the launcher. (Needs nvcc, not a GPU.)"""
    from semantic_aware_adaptive_kv_cache_precision_b200.ops._lib import plain_function
    for vocab in (1, 103, 18944, 18945, 50257, 151936):
        for sms in (1, 148):
            rows = plain_function("sakv_logprob_split_rows")(vocab, sms)
            assert 104 <= rows <= 128 and rows % 8 == 0
    for rows in (1, 32, 33, 128, 129, 185, 2047, 4097):
        padded = plain_function("sakv_logprob_split_tokens")(rows)
        tiles = -(-rows // 96)
        assert rows <= padded < rows + 32 * tiles and padded % (32 * tiles) == 0 and padded // tiles <= 96
    assert plain_function("sakv_logprob_split_tokens")(0) == 0
    assert plain_function("sakv_logprob_split_tokens")(2 ** 31 - 1) == 0 == plain_function("sakv_logprob_split_rows")(0, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [1024, 1032, 2056, 3136])
@pytest.mark.parametrize("rows", [5, 40, 96, 97, 256, 300, 352, 353, 520, 610])
def test_sums_in_several_chunks(rows, k):
    check(rows, k, 1333, torch.bfloat16, torch.float32 if rows % 2 else None, 0.5 if rows % 3 else 1.0,
          20.0 if rows % 5 == 0 else 0.0, seed=rows + k)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [40, 256])
def test_long_sums_of_16_bits(rows):
    """Numbers of one sign, where what is cut off adds up."""
    k = 4096
    g = torch.Generator(device="cuda").manual_seed(3)
    x = (torch.rand((rows, k), generator=g, device="cuda") + 0.5).to(torch.bfloat16)
    w = ((torch.rand((700, k), generator=g, device="cuda") + 0.5) / k).to(torch.bfloat16)
    targets = torch.randint(0, 700, (rows,), generator=g, device="cuda", dtype=torch.int32)
    got, lse = ops.token_logprobs(x, w, targets)
    z = x.double() @ w.double().t()
    want_lse = torch.logsumexp(z, 1)
    want = z.gather(1, targets.long()[:, None])[:, 0] - want_lse
    # 1,024 products and 64 additions on the tensor cores, each cut by a step of the sum (2^-23) at most, then three
    # additions that round by 2^-24; lse's own sum as above
    dz = (1024 + 64 + 2) * 2.0 ** -23 * z.amax()
    assert ((lse.double() - want_lse).abs() <= dz + 512 * 2.0 ** -23 + 2.0 ** -21 * (1 + want_lse)).all()
    assert ((got.double() - want).abs() <= 2 * dz + 512 * 2.0 ** -23 + 2.0 ** -21 * (2 + want_lse)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, k", [(torch.float32, 260), (torch.float32, 1028), (torch.bfloat16, 2056)])
def test_two_streams_and_graphs_at_once(dtype, k):
    """Calls side by side, and two captured calls replayed side by side, share nothing."""
    g = torch.Generator(device="cuda").manual_seed(5)
    sides = []
    for rows, vocab in ((70, 30000), (130, 9000)):
        x = torch.randn((rows, k), generator=g, device="cuda").to(dtype)
        w = (torch.randn((vocab, k), generator=g, device="cuda") / math.sqrt(k)).to(dtype)
        targets = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
        sides.append((x, w, targets, torch.cuda.Stream()))
    alone = [ops.token_logprobs(x, w, t)[0].clone() for x, w, t, _ in sides]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (x, w, t, stream) in enumerate(sides):
            with torch.cuda.stream(stream):
                got[i].append(ops.token_logprobs(x, w, t)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, many in zip(alone, got) for b in many)
    graphs = []
    for x, w, t, _ in sides:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = ops.token_logprobs(x, w, t)[0]
        graphs.append((graph, held))
    for x, _, _, _ in sides:
        x.copy_(x.flip(0))
    fresh = [ops.token_logprobs(x, w, t)[0] for x, w, t, _ in sides]
    torch.cuda.synchronize()
    for _ in range(3):
        for (graph, _), (_, _, _, stream) in zip(graphs, sides):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(held, want) for (_, held), want in zip(graphs, fresh))
    assert not torch.equal(fresh[0], alone[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, k, most", [(torch.bfloat16, 136, 256), (torch.bfloat16, 136, 512), (torch.float32, 131, 29),
                                            (torch.float32, 132, 29)])
def test_scratch_has_a_bound(monkeypatch, dtype, k, most):
    """Many rows are taken some at a time, so that what tiles leave stays below a bound, whichever way they go."""
    x, w, targets, got, lse = check(1301, k, 3001, dtype, seed=8)
    launches = []
    real = logprobs.call
    monkeypatch.setattr(logprobs, "call", lambda name, *args: (launches.append((name, args[3])), real(name, *args)))
    ops.token_logprobs(x, w, targets)
    assert len(launches) == 1
    # (tiles of the head: 16 of 192 rows, 24 of 128, 29 of 104)
    monkeypatch.setattr(logprobs, "SPLIT_PAIRS", most * (16 if dtype == torch.bfloat16 else 24 if k % 4 else 29))
    del launches[:]
    again, lse2 = ops.token_logprobs(x, w, targets)
    assert len(launches) >= 1301 // most and all(rows <= most for _, rows in launches), launches
    assert sum(rows for _, rows in launches) == 1301
    want, want_lse, bound = reference(x, w, targets, None, 1.0, 0.0)
    assert ((again.double() - want).abs() <= bound).all() and ((lse2.double() - want_lse).abs() <= bound).all()
    if dtype == torch.float32:
        assert torch.equal(again, got) and torch.equal(lse, lse2)


@pytest.mark.parametrize("rows", [5, 300])
def test_tiles_of_heads_as_long_as_numbers_go(rows):
    """Host code of the launcher: right up to where row numbers would leave 32 bits, refused from there on."""
    import ctypes
    from semantic_aware_adaptive_kv_cache_precision_b200.ops._lib import plain_function
    shape = (ctypes.c_int * 4)()
    for pairs in (1, 74, 1000):
        most = 2 ** 31 - 1 - 512 * pairs
        assert plain_function("sakv_logprob_shape")(rows, most, 64, pairs, shape) == 0
        full, height, tiles, launched = shape
        assert 1 <= height <= 128 and launched == pairs and (tiles - 1) * 2 * height < most <= tiles * 2 * height
        assert plain_function("sakv_logprob_shape")(rows, most + 1, 64, pairs, shape) != 0
    assert plain_function("sakv_logprob_shape")(rows, 1000, 64, 2 ** 20, shape) != 0


def test_caps_and_scales_that_32_bits_do_not_hold_are_refused():
    x, w, t = torch.zeros(3, 16), torch.zeros(50, 16), torch.zeros(3, dtype=torch.int32)
    for how in ({"softcap": 1e39}, {"softcap": 1e-39}, {"softcap": 1e-50}, {"scale": 1e39}, {"scale": -math.inf},
                {"scale": math.nan}):
        with pytest.raises(KernelError, match="softcap must be 0 or"):
            ops.token_logprobs(x, w, t, **how)
    for how in ({"softcap": 1e30}, {"softcap": 1e-30}, {"scale": -1e30}, {"scale": 0.0}):
        with pytest.raises(KernelError, match="CUDA device only"):
            ops.token_logprobs(x, w, t, **how)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_largest_and_smallest_caps(dtype):
    for rows in (5, 300):
        check(rows, 64, 700, dtype, softcap=1e4)
        x, w, targets, got, lse = check(rows, 64, 700, dtype)
        again, lse2 = ops.token_logprobs(x, w, targets, softcap=1e30)
        # (a cap that far away changes a logit by its last digit: two roundings of 2^-24, as near the cap as far from it)
        assert ((again - got).abs() <= 2.0 ** -19 * (1 + lse.abs() + got.abs())).all()
        low, lse3 = ops.token_logprobs(x, w, targets, softcap=1e-30)
        assert ((lse3 - math.log(700)).abs() <= 1e-5).all() and ((low + math.log(700)).abs() <= 1e-5).all()
        flat, _ = ops.token_logprobs(x, w, targets, scale=0.0)
        assert ((flat + math.log(700)).abs() <= 1e-5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 70, 300, 700])
@pytest.mark.parametrize("k, x_pad, head_at", [(37, 0, 0), (64, 3, 0), (64, 0, 1), (40, 24, 4), (1, 0, 0), (1031, 2, 3)])
def test_rows_that_are_copied_use_the_kernel(monkeypatch, rows, k, x_pad, head_at):
    """bfloat16 rows that TMA cannot take: no product of a library, whole and in pieces of the head and of the rows."""
    def none(*args, **how):
        raise AssertionError("a library's product")

    vocab = 1777
    g = torch.Generator(device="cuda").manual_seed(k + rows)
    x = torch.randn((rows, k + x_pad), generator=g, device="cuda").to(torch.bfloat16)[:, :k]
    flat = (torch.randn(vocab * k + head_at, generator=g, device="cuda") * 2 / math.sqrt(k)).to(torch.bfloat16)
    w = flat[head_at:].view(vocab, k)
    bias = torch.randn(vocab, generator=g, device="cuda")
    bias[:500] = -math.inf                                       # whole pieces of the head
    targets = torch.randint(500, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    targets[0], targets[1], targets[2] = 499, -1, vocab
    with monkeypatch.context() as m:
        for name in ("mm", "addmm", "matmul", "bmm"):
            m.setattr(torch, name, none)
        calls = [ops.token_logprobs(x, w, targets, bias, scale=0.5)]
        m.setattr(logprobs, "PIECE_ELEMENTS", 500 * (-(-k // 8) * 8))
        calls.append(ops.token_logprobs(x, w, targets, bias, scale=0.5))
        m.setattr(logprobs, "PIECE_ROWS", 250)
        m.setattr(logprobs, "SPLIT_PAIRS", 256 * 2)
        calls.append(ops.token_logprobs(x, w, targets, bias, scale=0.5))
    want, want_lse, bound = reference(x, w, targets, bias, 0.5, 0.0)
    bound = bound + 2.0 ** -21 * (1 + want_lse.abs())           # (pieces' sums are joined through a second logarithm)
    for got, lse in calls:
        assert ((lse.double() - want_lse).abs() <= bound).all(), ((lse.double() - want_lse).abs() / bound).max()
        assert ((got.double() - want).abs() <= bound)[3:].all()
        assert got[0] == -math.inf and got[1] == 0 and got[2].isnan()
    bias[:] = -math.inf
    monkeypatch.setattr(logprobs, "PIECE_ELEMENTS", 500 * (-(-k // 8) * 8))
    got, lse = ops.token_logprobs(x, w, targets, bias)
    assert (lse == -math.inf).all() and got[1] == 0 and got[[0] + list(range(2, rows))].isnan().all()
    x[1], bias[:] = math.nan, 0.0
    got, lse = ops.token_logprobs(x, w, targets, bias)
    assert lse[1].isnan() and torch.isfinite(lse[2:]).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held, _ = ops.token_logprobs(x, w, targets, bias)
    graph.replay()
    assert torch.equal(held[3:], got[3:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("k", [64, 63, 1100, 1101])
@pytest.mark.parametrize("rows", [7, 300])
def test_infinities_in_rows_and_in_the_head(dtype, k, rows):
    """As the formula has them, whichever way the rows go: a logit of -inf counts for nothing, one that is +inf or NaN makes
    its row NaN."""
    g = torch.Generator(device="cuda").manual_seed(k)
    x = torch.randn((rows, k), generator=g, device="cuda").to(dtype)
    w = torch.randn((700, k), generator=g, device="cuda").div_(math.sqrt(k)).to(dtype)
    x[:, 3] = x[:, 3].abs() + 0.5
    x[3, 3] = -1.0                           # its logit of the head's third row is +inf
    x[4, 3] = 0.0                            # and of this row NaN
    w[2, 3] = w[650, 3] = -math.inf
    x[5, 9], w[:, 9] = -math.inf, w[:, 9].abs() + 0.25          # every logit of this row is -inf, but for one
    w[77, 9] = -1.0                                             # that is +inf
    x[6, 1] = math.nan
    targets = torch.arange(rows, dtype=torch.int32, device="cuda")
    targets[1] = 650
    got, lse = ops.token_logprobs(x, w, targets)
    good = [0, 1, 2] + list(range(7, rows))
    assert got[3:7].isnan().all() and lse[3:7].isnan().all()
    kept = torch.ones(700, dtype=torch.bool, device="cuda")
    kept[[2, 650]] = False
    near = targets.clone()
    near[1], near[2] = 0, 0
    place = torch.cumsum(kept, 0).int() - 1                      # of a token among those that count
    want, want_lse, bound = reference(x[good], w[kept], place[near.long().clamp(max=699)][good], None, 1.0, 0.0)
    assert ((lse[good].double() - want_lse).abs() <= bound).all()
    assert got[1] == -math.inf and got[2] == -math.inf
    assert ((got[good].double() - want).abs() <= bound)[[0] + list(range(3, len(good)))].all()


@pytest.mark.gpu
def test_pieces_of_the_head_take_their_rows_in_one_launch(monkeypatch):
    """Where what the last rows leave takes a piece's scratch past its bound by some pairs."""
    monkeypatch.setattr(logprobs, "PIECE_ROWS", 250)
    monkeypatch.setattr(logprobs, "SPLIT_PAIRS", 2048)
    check(864, 37, 900, torch.bfloat16, torch.float32)

"""Logits under a decoder's rules, and the tokens chosen from them, against a plain loop in 64 bits.

The rules take at most five f32 steps on a value (penalty, product with the count, two differences,
the bias), each off by half a step, 2^-24, of a result no larger than
M = |l| max(theta, 1 / theta) + |f n| + |p| + sum |b|, and a token's biases as many steps as it has entries: the
bound on a value is (5 + entries) 2^-24 M, plus half a step of the output type relative to the value
(f16 below 2^-14: 2^-25). A log-probability adds, to the values' own error, that of log sum e^x: an
exponential's argument is rounded twice (2^-23 of at most 100 here, e^-100 and less being lost below
the sum), its instruction is off by 2^-22, and up to 2^7 sums follow one another within a thread
and in the merges (2^-24 each): 100 * 2^-23 + 2^-22 + 2^-17 < 2e-5, and half a step of the
result and of log and differences (values up to 64: 3 * 2^-18 more)."""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def types():
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def make(rows, vocab, dtype, history=0, biases=0, states=0, seed=0, ld=None, offset=0):
    """Logits (with rows ld apart, `offset` elements into their buffer) and a LogitRules."""
    import torch
    from telmo_b200 import LogitRules
    g = torch.Generator().manual_seed(seed)
    ld = ld or vocab
    store = (torch.randn(offset + rows * ld + 16, generator=g) * 3).to(types()[dtype]).cuda()
    logits = store[offset:offset + rows * ld].view(rows, ld)
    r = LogitRules()
    if history:
        # Many repeats, tokens outside the vocabulary among them, lengths from none to all.
        h = torch.randint(-2, max(2, min(vocab + 2, history)), (rows, history), generator=g, dtype=torch.int32)
        h[:, ::3] = torch.randint(0, vocab, (rows, len(range(0, history, 3))), generator=g, dtype=torch.int32)
        n = torch.randint(0, history + 1, (rows,), generator=g, dtype=torch.int32)
        n[0] = history
        if rows > 2:
            n[1], n[2] = 0, history + 50  # held to the width
        r.history, r.history_len = h.cuda(), n.cuda()
        r.repetition = (0.7 + torch.rand(rows, generator=g)).cuda()
        r.frequency = (torch.rand(rows, generator=g) - 0.3).cuda()
        r.presence = (torch.rand(rows, generator=g) - 0.3).cuda()
    if biases:
        ids = torch.randint(-1, vocab + 1, (rows, biases), generator=g, dtype=torch.int32)
        ids[:, : biases // 4] = ids[:, -1:]  # one token many times
        b = torch.randn((rows, biases), generator=g) * 4
        b[rows // 2, biases // 2] = -math.inf
        r.bias_ids, r.bias = ids.cuda(), b.cuda()
    if states:
        words = -(-vocab // 32)
        m = torch.randint(-2 ** 31, 2 ** 31, (states, words), generator=g, dtype=torch.int64).int()
        m[0] = 0
        if states > 1:
            m[1] = 0
            m[1, (vocab - 1) // 32] = -2 ** 31 if (vocab - 1) % 32 == 31 else 1 << ((vocab - 1) % 32)
        st = torch.arange(rows, dtype=torch.int32) % (states + 2) - 1  # without a mask ... out of range
        r.allowed, r.state = m.cuda(), st.cuda()
    return logits, r


def host(t):
    return None if t is None else t.cpu().numpy()


def values(logits, vocab, r):
    """The rules in 64 bits, and the bound on a value's f32 error."""
    x = logits[:, :vocab].double().cpu().numpy().copy()
    tol = np.zeros_like(x)
    h, n, th, fr, pr = (host(t) for t in (r.history, r.history_len, r.repetition, r.frequency, r.presence))
    bi, bv, al, st = (host(t) for t in (r.bias_ids, r.bias, r.allowed, r.state))
    rows = x.shape[0]
    for row in range(rows):
        size, steps = np.abs(x[row]), np.zeros(vocab)
        if h is not None:
            said = h[row, : max(0, min(int(n[row]), h.shape[1]))]
            said = said[(said >= 0) & (said < vocab)]
            c = np.bincount(said, minlength=vocab)
            at = c > 0
            t = float(th[row]) if th is not None else 1.0
            f = float(fr[row]) if fr is not None else 0.0
            p = float(pr[row]) if pr is not None else 0.0
            v = np.where(x[row] > 0, x[row] / t, x[row] * t) - f * c - p
            x[row] = np.where(at, v, x[row])
            size = np.where(at, size * max(t, 1 / t) + abs(f) * c + abs(p), size)
            steps += 5 * at
        if bi is not None:
            for tok, b in zip(bi[row], bv[row].astype(np.float64)):
                if 0 <= tok < vocab:
                    x[row, tok] += b
                    size[tok] += abs(b) if np.isfinite(b) else 0
                    steps[tok] += 1 + (steps[tok] == 0)
        if al is not None:
            s = int(st[row]) if st is not None else row
            if s >= al.shape[0]:
                x[row] = -np.inf
            elif s >= 0:
                tok = np.arange(vocab)
                x[row, ((al[s].astype(np.int64)[tok // 32] >> (tok % 32)) & 1) == 0] = -np.inf
        tol[row] = steps * 2.0 ** -24 * np.where(np.isfinite(size), size, 0)
    return x, tol


def check_constrain(ctx, rows, vocab, dtype, ld=None, out_ld=None, offset=0, out_offset=0, in_place=False, stream=None,
                    **more):
    import torch
    from telmo_b200 import Kernels
    logits, r = make(rows, vocab, dtype, ld=ld, offset=offset, **more)
    ld = ld or vocab
    out_ld = ld if in_place else out_ld or vocab
    x, tol = values(logits, vocab, r)
    if in_place:
        out = logits
    else:
        out = torch.full((out_offset + rows * out_ld,), 7.0, device="cuda").to(logits.dtype)[out_offset:].view(rows, out_ld)
    before = out.clone()
    Kernels(ctx).constrain_logits(logits, ld, rows, vocab, r, out, out_ld, stream=stream)
    ctx.check(stream)
    got = out[:, :vocab].double().cpu().numpy()
    assert np.array_equal(np.isinf(got), np.isinf(x)) and not np.isnan(got).any()
    fin = np.isfinite(x)
    assert (got[~fin] == x[~fin]).all()
    lim = tol + (np.abs(np.where(fin, x, 0)) + tol) * HALF[dtype] * (dtype != "f32") + (2.0 ** -25 if dtype == "f16" else 0)
    off = np.abs(got[fin] - x[fin])
    assert (off <= lim[fin]).all(), float((off - lim[fin]).max())
    assert torch.equal(out[:, vocab:], before[:, vocab:])


def check_choose(ctx, rows, vocab, dtype, k, ld=None, offset=0, stream=None, logits=None, r=None, **more):
    import torch
    from telmo_b200 import Kernels
    if logits is None:
        logits, r = make(rows, vocab, dtype, ld=ld, offset=offset, **more)
    x, tol = values(logits, vocab, r)
    ids = torch.full((rows + 1, k), 77, dtype=torch.int32, device="cuda")
    lp = torch.full((rows + 1, k), 77.0, device="cuda")
    Kernels(ctx).choose_tokens(logits, ld or vocab, rows, vocab, r, k, ids, lp, stream=stream)
    ctx.check(stream)
    assert (ids[rows] == 77).all() and (lp[rows] == 77).all()
    got, glp = ids[:rows].cpu().numpy(), lp[:rows].double().cpu().numpy()
    for row in range(rows):
        left = int((x[row] > -np.inf).sum())
        order = np.argsort(-x[row], kind="stable")[:k]
        n = min(k, left)
        assert (got[row, n:] == -1).all() and (glp[row, n:] == -np.inf).all()
        if not n:
            continue
        assert len(set(got[row, :n])) == n and (got[row, :n] >= 0).all()
        top = x[row].max()
        lse = top + np.log(np.exp(x[row] - top).sum())
        for j in range(n):
            a, b = got[row, j], order[j]
            # The same token, or one whose value is within the values' own f32 error of it; where
            # no value has an error, exactly the lowest of those that tie.
            assert a == b or (tol[row, a] + tol[row, b] > 0 and abs(x[row, a] - x[row, b]) <= tol[row, a] + tol[row, b])
            assert abs(glp[row, j] - (x[row, a] - lse)) <= 3.2e-5 + 2 * tol[row].max()


SIZES = [(1, 1), (1, 2), (3, 7), (2, 31), (5, 32), (4, 33), (7, 257), (3, 2049), (2, 8191), (2, 8192), (3, 8193),
         (1, 16385), (9, 8198), (1, 49157), (2, 70001), (300, 97)]


@pytest.mark.parametrize("rows,vocab", SIZES)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_constrain_sizes(ctx, rows, vocab, dtype):
    check_constrain(ctx, rows, vocab, dtype, history=40, biases=9, states=4, seed=vocab)


@pytest.mark.parametrize("rows,vocab", SIZES)
@pytest.mark.parametrize("dtype,k", [("f32", 1), ("bf16", 2), ("f16", 3), ("f32", 4), ("bf16", 5), ("f32", 8)])
def test_choose_sizes(ctx, rows, vocab, dtype, k):
    check_choose(ctx, rows, vocab, dtype, k, history=40, biases=9, states=4, seed=vocab)


@pytest.mark.parametrize("history,biases,states", [(0, 0, 0), (1, 0, 0), (700, 0, 0), (3000, 0, 0), (0, 1, 0), (0, 40, 0),
                                                   (0, 300, 0), (0, 0, 1), (0, 0, 5), (64, 33, 0), (64, 0, 2), (0, 31, 2)])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_each_rule(ctx, history, biases, states, dtype):
    check_constrain(ctx, 6, 9001, dtype, history=history, biases=biases, states=states, seed=3)
    check_choose(ctx, 6, 9001, dtype, 4, history=history, biases=biases, states=states, seed=3)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("ld,out_ld,offset,out_offset", [(1000, 1000, 1, 1), (1001, 1000, 0, 0), (1003, 1001, 3, 5),
                                                         (1008, 1008, 8, 0), (1024, 999, 7, 2)])
def test_strides_and_alignment(ctx, dtype, ld, out_ld, offset, out_offset):
    check_constrain(ctx, 5, 999, dtype, ld=ld, out_ld=out_ld, offset=offset, out_offset=out_offset, history=30, biases=5,
                    states=3, seed=1)
    check_constrain(ctx, 5, 999, dtype, ld=ld, offset=offset, in_place=True, history=30, biases=5, states=3, seed=1)
    check_choose(ctx, 5, 999, dtype, 4, ld=ld, offset=offset, history=30, biases=5, states=3, seed=1)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [9, 500, 20000, 100000])
def test_ties_go_to_the_lowest_token(ctx, dtype, vocab):
    """Values from a handful: nearly every choice is a tie."""
    import torch
    from telmo_b200 import LogitRules
    logits = torch.randint(0, 3, (4, vocab), generator=torch.Generator().manual_seed(vocab)).to(types()[dtype]).cuda()
    logits[1] = 0
    logits[2, ::2] = -0.0
    check_choose(ctx, 4, vocab, dtype, 8, logits=logits, r=LogitRules())


@pytest.mark.parametrize("vocab", [10, 2049, 40000])
def test_infinities_and_nans(ctx, vocab):
    """Masked places may hold anything; -infinity is never chosen; NaN and +infinity where allowed."""
    import torch
    from telmo_b200 import Kernels, LogitRules
    logits = torch.randn((6, vocab), generator=torch.Generator().manual_seed(1)).cuda()
    words = -(-vocab // 32)
    mask = torch.full((1, words), -1, dtype=torch.int32, device="cuda")
    mask[0, 0] = ~0b110
    state = torch.zeros(6, dtype=torch.int32, device="cuda")
    logits[0, 1], logits[0, 2] = math.nan, math.inf  # masked
    logits[1] = -math.inf
    logits[2, 3:] = torch.finfo(torch.float32).min
    logits[2, 0] = torch.finfo(torch.float32).min
    logits[3, 5] = math.nan
    logits[4, 6] = math.inf
    r = LogitRules(allowed=mask, state=state)
    ids = torch.zeros((6, 2), dtype=torch.int32, device="cuda")
    lp = torch.zeros((6, 2), device="cuda")
    out = torch.empty_like(logits)
    k = Kernels(ctx)
    k.choose_tokens(logits, vocab, 6, vocab, r, 2, ids, lp)
    k.constrain_logits(logits, vocab, 6, vocab, r, out, vocab)
    ctx.check()
    assert (out[:, 1:3] == -math.inf).all()
    keep = torch.ones(vocab, dtype=torch.bool, device="cuda")
    keep[1:3] = False
    assert torch.equal(out[:, keep].view(torch.int32), logits[:, keep].view(torch.int32))
    x = logits[:, keep]
    tok = torch.arange(vocab, device="cuda")[keep]
    for row in (0, 5):
        assert ids[row].tolist() == tok[torch.topk(x[row], 2).indices].tolist()
        want = torch.topk(x[row].double(), 2).values - torch.logsumexp(x[row].double(), 0)
        assert (lp[row].double() - want).abs().max() <= 3.2e-5
    assert ids[1].tolist() == [-1, -1] and (lp[1] == -math.inf).all()
    assert ids[2].tolist() == [0, 3]
    assert (lp[2] + math.log(vocab - 2)).abs().max() <= 3.2e-5
    assert ids[3, 0].item() == tok[torch.nan_to_num(x[3], nan=-math.inf).argmax()].item() and lp[3].isnan().all()
    assert ids[4, 0].item() == 6 and lp[4].isnan().all()


def test_rules_that_are_empty(ctx):
    """No rules, rules of no entries, no rows."""
    import torch
    from telmo_b200 import Kernels, LogitRules
    k = Kernels(ctx)
    logits = torch.randn((3, 100), device="cuda")
    empty = torch.empty((3, 0), device="cuda")
    none = LogitRules(history=empty.int(), history_len=torch.zeros(3, dtype=torch.int32, device="cuda"),
                      repetition=torch.ones(3, device="cuda"), bias_ids=empty.int(), bias=empty)
    for r in (None, LogitRules(), none):
        out = torch.empty_like(logits)
        k.constrain_logits(logits, 100, 3, 100, r, out, 100)
        ids = torch.empty((3, 1), dtype=torch.int32, device="cuda")
        k.choose_tokens(logits, 100, 3, 100, r, 1, ids)
        ctx.check()
        assert torch.equal(out, logits) and torch.equal(ids[:, 0].long(), logits.argmax(1))
    k.constrain_logits(logits, 100, 0, 100, None, out, 100)
    k.choose_tokens(logits, 100, 0, 100, None, 1, ids)
    ctx.check()


def test_views_of_larger_buffers(ctx):
    """Lists and masks that are the first columns of wider matrices; masks by row without states."""
    import torch
    from telmo_b200 import LogitRules
    logits, r = make(4, 300, "f32", history=50, biases=20, states=4, seed=8)

    def wide(t, fill):
        w = torch.full((t.shape[0], t.shape[1] + 13), fill, dtype=t.dtype, device="cuda")
        w[:, : t.shape[1]] = t
        return w[:, : t.shape[1]]
    check_choose(ctx, 4, 300, "f32", 3, logits=logits, r=LogitRules(
        history=wide(r.history, 5), history_len=r.history_len, frequency=r.frequency, bias_ids=wide(r.bias_ids, 6),
        bias=wide(r.bias, 50.0), allowed=wide(r.allowed, -1)))


def test_many_rows(ctx):
    """More rows than one grid's second dimension holds, each with rules of its own."""
    check_choose(ctx, 70001, 3, "f32", 2, history=4, biases=2, states=3, seed=2)
    check_constrain(ctx, 70001, 3, "bf16", history=4, biases=2, states=3, seed=2)


def test_a_bias_for_every_token(ctx):
    """Lists as long as the vocabulary, tokens among them twice and many times: time for those alone."""
    check_constrain(ctx, 2, 20000, "f32", history=40, biases=20000, states=3, seed=6)
    check_choose(ctx, 2, 20000, "bf16", 4, history=40, biases=20000, states=3, seed=6)


def test_too_many_biases_are_refused(ctx):
    import torch
    from telmo_b200 import Kernels, LogitRules, TelmoError
    x, most = torch.zeros((1, 10), device="cuda"), 1 << 20
    ids, bias = torch.full((1, most + 1), 3, dtype=torch.int32, device="cuda"), torch.zeros((1, most + 1), device="cuda")
    bias[0, most - 1] = 2.5
    for call in (lambda r: Kernels(ctx).constrain_logits(x, 10, 1, 10, r, x, 10),
                 lambda r: Kernels(ctx).choose_tokens(x, 10, 1, 10, r, 1, ids)):
        with pytest.raises(TelmoError):
            call(LogitRules(bias_ids=ids, bias=bias))
    Kernels(ctx).constrain_logits(x, 10, 1, 10, LogitRules(bias_ids=ids[:, :most], bias=bias[:, :most]), x, 10)
    ctx.check()
    assert x.tolist() == [[0, 0, 0, 2.5, 0, 0, 0, 0, 0, 0]]


@pytest.mark.parametrize("times", [1, 2, 5])
def test_biases_of_tokens_that_stand_several_times(ctx, times):
    """Every token `times` times, some once more, one many times, in mixed order."""
    import torch
    from telmo_b200 import LogitRules
    vocab, g = 5000, torch.Generator().manual_seed(9)
    ids = torch.cat([torch.arange(vocab).repeat(times), torch.arange(0, vocab, 7), torch.full((300,), 77)])
    ids = torch.stack([ids[torch.randperm(len(ids), generator=g)] for _ in range(3)]).int()
    bias = torch.randn(ids.shape, generator=g)
    logits = torch.randn((3, vocab), generator=g).cuda()
    r = LogitRules(bias_ids=ids.cuda(), bias=bias.cuda())
    check_choose(ctx, 3, vocab, "f32", 8, logits=logits, r=r)
    from telmo_b200 import Kernels
    x, tol = values(logits, vocab, r)
    out = torch.empty_like(logits)
    Kernels(ctx).constrain_logits(logits, vocab, 3, vocab, r, out, vocab)
    ctx.check()
    assert (np.abs(out.double().cpu().numpy() - x) <= tol).all()


@pytest.mark.parametrize("tokens,times", [(2, 3), (40, 3), (33, 40), (64, 300), (700, 30), (5000, 20), (64, 16384), (1, 1 << 20)])
@pytest.mark.parametrize("order", ["mixed", "in turn", "in runs"])
def test_some_tokens_very_many_times(ctx, tokens, times, order):
    """Biases of each token add up one after another, in list order: the very bits of that. The longest lists take
    milliseconds (2^20 entries are read a bounded number of times, not once for each time a token stands there)."""
    import torch
    from telmo_b200 import Kernels, LogitRules
    vocab, g = 9000, np.random.default_rng(tokens)
    names = g.permutation(vocab)[:tokens]
    ids = np.repeat(names, times) if order == "in runs" else np.tile(names, times)
    if order == "mixed":
        ids = g.permutation(ids)
    bias = g.standard_normal(len(ids)).astype(np.float32)
    x = g.standard_normal((1, vocab)).astype(np.float32)
    want = x.copy()
    for v in names:
        want[0, v] += np.cumsum(bias[ids == v], dtype=np.float32)[-1]
    r = LogitRules(bias_ids=torch.from_numpy(ids.astype(np.int32))[None].cuda(), bias=torch.from_numpy(bias)[None].cuda())
    logits = torch.from_numpy(x).cuda()
    out, best = torch.empty_like(logits), torch.zeros((1, 4), dtype=torch.int32, device="cuda")
    k = Kernels(ctx)
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    k.constrain_logits(logits, vocab, 1, vocab, None, out, vocab)  # the kernels are loaded before the clock runs
    k.choose_tokens(logits, vocab, 1, vocab, None, 4, best)
    begin.record()
    k.constrain_logits(logits, vocab, 1, vocab, r, out, vocab)
    k.choose_tokens(logits, vocab, 1, vocab, r, 4, best)
    end.record()
    ctx.check()
    assert np.array_equal(out.cpu().numpy().view(np.int32), want.view(np.int32))
    assert best[0].tolist() == np.argsort(-want[0], kind="stable")[:4].tolist()
    assert begin.elapsed_time(end) < 200  # ms


@pytest.mark.parametrize("rows,vocab,history,biases", [(3, 9001, 9000, 2500), (2, 40000, 30000, 3000), (500, 33000, 9000, 0),
                                                       (200, 65540, 12000, 0)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_more_listed_tokens_than_numbers(ctx, rows, vocab, history, biases, dtype):
    """Thousands of listed tokens in every window, which are numbered 2048 at a time. (Where one block has a row of
    65540, a thread adds up to 150 values: 150 2^-24 in place of 2^-17 adds 1.4e-6 to the bound on a log-probability;
    the values' own bound, at least 2 * 5 * 2^-24 * 4 there, covers it.)"""
    check_constrain(ctx, rows, vocab, dtype, history=history, biases=biases, states=3, seed=5)
    check_choose(ctx, rows, vocab, dtype, 5, history=history, biases=biases, states=3, seed=5)


def test_offsets_beyond_32_bits(ctx):
    """Rows whose offsets pass 2^31 elements."""
    import torch
    from telmo_b200 import Kernels
    ld = (1 << 30) + 3
    store = torch.zeros(2 * ld + 100, dtype=torch.bfloat16, device="cuda")
    store[2 * ld + 42] = 5
    ids = torch.zeros((3, 1), dtype=torch.int32, device="cuda")
    k = Kernels(ctx)
    k.choose_tokens(store, ld, 3, 100, None, 1, ids)
    k.constrain_logits(store, ld, 3, 100, None, store, ld)
    ctx.check()
    assert ids[:, 0].tolist() == [0, 0, 42] and store[2 * ld + 42] == 5


def test_the_largest_vocabulary(ctx):
    """2^30 tokens, the last of them listed."""
    import torch
    from telmo_b200 import Kernels, LogitRules, TelmoError
    v = 1 << 30
    store = torch.zeros(v + 1, dtype=torch.bfloat16, device="cuda")
    store[0], store[v - 1], store[v] = 4, 8, 9
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    r = LogitRules(history=i32([[v - 1, v - 1]]), history_len=i32([2]), frequency=torch.tensor([1.5], device="cuda"))
    ids, k = i32([[0, 0]]), Kernels(ctx)
    k.choose_tokens(store, v, 1, v, r, 2, ids)
    k.constrain_logits(store, v, 1, v, r, store, v)
    ctx.check()
    assert ids.tolist() == [[v - 1, 0]]
    assert store[v - 1] == 5 and store[v] == 9 and store[0] == 4 and store[1:v - 1].count_nonzero() == 0
    with pytest.raises(TelmoError):
        k.choose_tokens(store, v + 1, 1, v + 1, None, 2, ids)


def test_streams_and_graphs(ctx):
    import torch
    from telmo_b200 import Kernels
    side = torch.cuda.Stream()
    check_choose(ctx, 5, 9000, "f32", 2, stream=side, history=50, biases=5, states=2, seed=4)
    check_constrain(ctx, 5, 9000, "f32", stream=side, history=50, biases=5, states=2, seed=4)
    k = Kernels(ctx)
    sets = [make(4, 40000, "f32", history=300, biases=20, states=3, seed=s) for s in (1, 2)]
    outs = [(torch.zeros((4, 2), dtype=torch.int32, device="cuda"), torch.zeros((4, 2), device="cuda"),
             torch.zeros((4, 40000), device="cuda")) for _ in range(4)]

    def both(i, o):
        k.choose_tokens(sets[i][0], 40000, 4, 40000, sets[i][1], 2, o[0], o[1])
        k.constrain_logits(sets[i][0], 40000, 4, 40000, sets[i][1], o[2], 40000)
    graphs = []
    for i in range(2):
        both(i, outs[i])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            both(i, outs[2 + i])
        graphs.append((g, torch.cuda.Stream()))
    for _ in range(3):
        for g, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], outs[2 + i]))


def test_columns_and_overlaps_are_refused(ctx):
    """Views whose elements are not where a row's are (a column to write tokens to, a column of parameters), and
    outputs that overlap the logits."""
    import torch
    from telmo_b200 import Kernels, LogitRules, TelmoError
    k = Kernels(ctx)
    store = torch.randn((4, 200), device="cuda")
    x, y = store[:, :100], store[:, 100:]
    i32 = dict(dtype=torch.int32, device="cuda")
    said, n, ids = torch.zeros((4, 9), **i32), torch.ones(4, **i32), torch.zeros((4, 1), **i32)
    table = torch.ones((4, 3), device="cuda")
    before = store.clone()
    for call in (lambda: k.choose_tokens(x, 200, 4, 100, None, 1, said[:, 3:4]),
                 lambda: k.choose_tokens(x, 200, 4, 100, None, 1, said[:, 3]),
                 lambda: k.choose_tokens(x, 200, 4, 100, None, 1, ids, store[:, 1:2]),
                 lambda: k.choose_tokens(x, 100, 4, 100, None, 1, ids),
                 lambda: k.choose_tokens(x, 200, 4, 101, None, 1, ids),
                 lambda: k.choose_tokens(x, 200, 4, 100, LogitRules(said, n, repetition=table[:, 1]), 1, ids),
                 lambda: k.choose_tokens(x, 200, 4, 100, LogitRules(said, n, presence=table[:, :1]), 1, ids),
                 lambda: k.choose_tokens(x, 200, 4, 100, LogitRules(said, said[:, 0]), 1, ids),
                 lambda: k.constrain_logits(store, 200, 4, 100, None, store, 150),
                 lambda: k.constrain_logits(store, 200, 4, 100, None, store[0, 50:], 200),
                 lambda: k.constrain_logits(store[0, 50:], 200, 3, 100, None, store, 200),
                 lambda: k.constrain_logits(store, 200, 4, 100, None, store[1], 150)):
        with pytest.raises(TelmoError):
            call()
    ctx.check()
    assert torch.equal(store, before) and not said.any()
    k.constrain_logits(x, 200, 4, 100, None, y, 200)  # side by side
    k.constrain_logits(store, 200, 1, 100, None, store, 100)  # one row, in place
    ctx.check()
    assert torch.equal(y, before[:, :100]) and torch.equal(x, before[:, :100])


def test_refusals(ctx):
    import ctypes
    import torch
    from telmo_b200 import Kernels, LogitRules, TelmoError, _lib
    k = Kernels(ctx)
    x = torch.randn((4, 100), device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    ids, lp, out = torch.zeros((4, 2), **i32), torch.zeros((4, 2), device="cuda"), torch.full((4, 100), 3.0, device="cuda")
    h, n, f = torch.zeros((4, 5), **i32), torch.zeros(4, **i32), torch.ones(4, device="cuda")
    m = torch.zeros((4, 4), **i32)
    bad = [LogitRules(history=h), LogitRules(repetition=f), LogitRules(history=h[:3], history_len=n),
           LogitRules(history=h.long(), history_len=n), LogitRules(history=h, history_len=n.long()),
           LogitRules(history=h, history_len=n, repetition=f[:3]), LogitRules(history=h, history_len=n, frequency=f.double()),
           LogitRules(history=h.t(), history_len=n), LogitRules(history=h.cpu(), history_len=n),
           LogitRules(bias_ids=h), LogitRules(bias_ids=h, bias=torch.ones((4, 4), device="cuda")),
           LogitRules(bias_ids=h, bias=h), LogitRules(allowed=m[:, :3]), LogitRules(allowed=m[:3]), LogitRules(state=n),
           LogitRules(allowed=m.float()), LogitRules(allowed=m, state=n[:3]), LogitRules(allowed=m, state=n.cpu())]
    for r in bad:
        with pytest.raises(TelmoError):
            k.constrain_logits(x, 100, 4, 100, r, out, 100)
        with pytest.raises(TelmoError):
            k.choose_tokens(x, 100, 4, 100, r, 2, ids, lp)
    for call in (lambda: k.choose_tokens(x, 100, 4, 100, None, 0, ids), lambda: k.choose_tokens(x, 100, 4, 100, None, 9, ids),
                 lambda: k.choose_tokens(x, 100, 4, 100, None, 3, ids), lambda: k.choose_tokens(x, 99, 4, 100, None, 2, ids),
                 lambda: k.choose_tokens(x, 100, 5, 100, None, 1, ids), lambda: k.choose_tokens(x, 100, 4, 0, None, 1, ids),
                 lambda: k.choose_tokens(x.double(), 100, 4, 100, None, 1, ids),
                 lambda: k.choose_tokens(x, 100, 4, 100, None, 2, ids.long()),
                 lambda: k.choose_tokens(x, 100, 4, 100, None, 2, ids, lp.half()),
                 lambda: k.choose_tokens(x.cpu(), 100, 4, 100, None, 2, ids, lp),
                 lambda: k.constrain_logits(x, 100, 4, 100, None, out.half(), 100),
                 lambda: k.constrain_logits(x, 100, 4, 100, None, out, 99),
                 lambda: k.constrain_logits(x, 100, 4, 100, None, out[:3], 100)):
        with pytest.raises(TelmoError):
            call()
    L, arg, hd = _lib.load(), _lib.TELMO_ERR_ARGUMENT, ctx.handle
    px, po, pi = x.data_ptr(), out.data_ptr(), ids.data_ptr()

    def rules(**fields):
        r = _lib.LogitRules()
        for name, v in fields.items():
            setattr(r, name, v)
        return ctypes.byref(r)
    hp, np_, mp = h.data_ptr(), n.data_ptr(), m.data_ptr()
    for r in (rules(history=hp, n_history=5, history_ld=5), rules(frequency=f.data_ptr()),
              rules(history=hp, n_history=6, history_ld=5, history_len=np_),
              rules(history=hp + 2, n_history=5, history_ld=5, history_len=np_), rules(n_bias=2, bias_ld=2),
              rules(n_bias=2, bias_ld=1, bias_ids=hp, bias=hp), rules(allowed=mp, n_states=4, allowed_ld=3),
              rules(allowed=mp, n_states=3, allowed_ld=4), rules(allowed=mp, n_states=0, allowed_ld=4, state=np_),
              rules(state=np_)):
        assert L.telmo_logits_constrain(hd, px, 0, 100, 4, 100, r, po, 100, None) == arg
        assert L.telmo_logits_choose(hd, px, 0, 100, 4, 100, r, 2, pi, None, None) == arg
    assert L.telmo_logits_constrain(hd, px, 2, 100, 4, 100, None, po, 100, None) == arg
    assert L.telmo_logits_constrain(hd, px + 2, 0, 99, 4, 99, None, po, 100, None) == arg
    assert L.telmo_logits_constrain(hd, px, 0, 100, 4, 100, None, po + 1, 100, None) == arg
    assert L.telmo_logits_constrain(hd, None, 0, 100, 4, 100, None, po, 100, None) == arg
    assert L.telmo_logits_choose(hd, px, 0, 100, 4, 100, None, 2, None, None, None) == arg
    assert L.telmo_logits_choose(hd, px, 0, 100, 4, 100, None, 2, pi + 2, None, None) == arg
    assert L.telmo_logits_choose(None, px, 0, 100, 4, 100, None, 2, pi, None, None) == arg
    assert (out == 3).all()


@pytest.mark.parametrize("vocab", [700, 8192, 20011, 131072])
@pytest.mark.parametrize("k", [1, 3, 8])
def test_rows_in_order(ctx, vocab, k):
    """Rising rows, whose every tile holds larger values than all before, falling ones, rows that rise within tiles and
    from thread to thread, and one value alone: the bound of the choice rises at every step or never."""
    import torch
    from telmo_b200 import LogitRules
    v = torch.arange(vocab)
    rows = torch.stack([v, -v, v % 16 * 8192 + v // 16, (v % 8192) * 16 + v // 8192, torch.zeros(vocab, dtype=torch.int64)])
    check_choose(ctx, 5, vocab, "f32", k, logits=(rows.float() / vocab).cuda(), r=LogitRules())


@pytest.mark.parametrize("vocab", [33, 2049, 70001])
def test_masks_of_either_type(ctx, vocab):
    """32-bit words as torch.int32 or torch.uint32; the highest bit of a word is a token like the others."""
    import torch
    from telmo_b200 import Kernels, LogitRules
    k, words = Kernels(ctx), -(-vocab // 32)
    x = torch.randn((3, vocab), generator=torch.Generator().manual_seed(vocab)).cuda()
    masks = torch.randint(-2 ** 31, 2 ** 31, (3, words), generator=torch.Generator().manual_seed(1), dtype=torch.int64)
    masks[0] = 1 << 31
    got = []
    for m in (masks.to(torch.int32).cuda(), (masks & 0xffffffff).to(torch.uint32).cuda()):
        out, ids = torch.empty_like(x), torch.empty((3, 2), dtype=torch.int32, device="cuda")
        k.constrain_logits(x, vocab, 3, vocab, LogitRules(allowed=m), out, vocab)
        k.choose_tokens(x, vocab, 3, vocab, LogitRules(allowed=m), 2, ids)
        ctx.check()
        got.append((out, ids))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    allowed = torch.isfinite(got[0][0][0]).nonzero()[:, 0].cpu()
    assert allowed.tolist() == list(range(31, vocab, 32))

"""A decoding step of the three operators together: a 4-bit head's logits, a decoder's rules over them,
and the tokens chosen, in rows of a beam, several steps on end with the tokens so far growing."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab,width,dtype", [(1, 2049, 1024, "f32"), (5, 8198, 640, "f32"), (40, 3001, 512, "bf16")])
def test_steps(ctx, rows, vocab, width, dtype):
    import torch
    from telmo_b200 import Epilogue, Kernels, LogitRules, PackedWeights, Precision
    from test_logits_gpu import values
    kern = Kernels(ctx)
    g = np.random.default_rng(vocab)
    packed = PackedWeights.encode(g.standard_normal((vocab, width)).astype(np.float32) / np.sqrt(width), vocab, width,
                                  Precision.Q4, group=64, zeros=True)
    head = packed.upload(ctx)
    bias = torch.from_numpy(g.standard_normal(vocab).astype(np.float32)).cuda()
    hidden = torch.from_numpy(g.standard_normal((rows, width)).astype(np.float32)).cuda()
    if dtype == "bf16":
        hidden = hidden.bfloat16()
    steps, k = 6, 3
    history = torch.full((rows, steps), -1, dtype=torch.int32, device="cuda")
    length = torch.zeros(rows, dtype=torch.int32, device="cuda")
    words = -(-vocab // 32)
    # Even tokens after odd ones and the other way round: a grammar of two states.
    allowed = torch.empty((2, words), dtype=torch.int32, device="cuda")
    allowed[0], allowed[1] = 0x55555555, -0x55555556
    state = torch.zeros(rows, dtype=torch.int32, device="cuda")
    rules = LogitRules(history=history, history_len=length, frequency=torch.full((rows,), 0.5, device="cuda"),
                       repetition=torch.full((rows,), 1.5, device="cuda"), allowed=allowed, state=state)
    logits = torch.empty((rows, vocab), device="cuda")
    under = torch.empty_like(logits)
    ids, plain = (torch.empty((rows, k), dtype=torch.int32, device="cuda") for _ in range(2))
    lp, plain_lp = (torch.empty((rows, k), device="cuda") for _ in range(2))
    chosen = []
    for step in range(steps):
        kern.linear(hidden, rows, head, logits, Epilogue(bias=bias))
        kern.constrain_logits(logits, vocab, rows, vocab, rules, under, vocab)
        kern.choose_tokens(logits, vocab, rows, vocab, rules, k, ids, lp)
        # The same choice from the constrained logits, without rules.
        kern.choose_tokens(under, vocab, rows, vocab, None, k, plain, plain_lp)
        ctx.check()
        assert torch.equal(ids, plain) and torch.allclose(lp, plain_lp, rtol=0, atol=4e-5)
        x, tol = values(logits, vocab, rules)
        best = ids[:, 0].cpu().numpy()
        assert (best % 2 == step % 2).all()
        assert (x[np.arange(rows), best] >= x.max(axis=1) - 2 * tol.max(axis=1)).all()
        chosen.append(best)
        history[:, step] = ids[:, 0]
        length += 1
        state = rules.state = 1 - state
    # A penalised token comes again only where nothing better is left; six steps over thousands leave plenty.
    for row in np.stack(chosen, axis=1):
        assert len(set(row.tolist())) == steps
    head.free()

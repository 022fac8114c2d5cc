"""Attention where its arithmetic and its bounds end, against 64-bit forms."""
import pytest
import torch

import attention_reference as ref
from test_gpu_attention import Batch, eng, stream  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def test_more_tokens_than_the_bound(eng):  # noqa: F811
    """Of a sequence of more than `longest` tokens the first `longest` are computed, and all of the others' that keep to it; with
    more tiles of rows than a group finds by itself, and with fewer."""
    for sequences, longest, counts in ((1100, 1, {40: 4000}), (1100, 3, {0: 3000, 7: 500}), (700, 2, {699: 5000}), (30, 40, {3: 900})):
        print(f"{sequences} sequences, longest {longest}, {counts}", flush=True)
        of = [counts.get(b, 1 + b % longest) for b in range(sequences)]
        b = Batch(eng, "bf16", 32, 1, 16, 16, of, [n + 20 for n in of], seed=41)
        b.out.fill_(7.0)
        eng.attention(b.q, b.kc, b.vc, b.table, b.lengths, b.out, b.ws, starts=b.starts, longest=longest, stream=stream())
        torch.cuda.synchronize()
        first = torch.cat([b.starts[i] + torch.arange(min(n, longest), device="cuda") for i, n in enumerate(of)])
        # A token by itself: its sequence's keys up to its own.
        at = torch.cat([21 + torch.arange(min(n, longest)) for n in of])
        of_token = torch.cat([torch.full((min(n, longest),), i) for i, n in enumerate(of)]).cuda()
        want, bound, _ = ref.attention(b.q[first], b.kc, b.vc, b.table[of_token], at, [1] * len(at), 32, 0.25, True, 0)
        got = b.out[first].cpu().double()
        assert ((got - want).abs() <= bound + ref.half_step(torch.bfloat16) * (want.abs() + bound)).all()
        assert (b.out[b.n:] == 7).all()

"""Log probabilities at the far ends of what the call takes, against 64 bits."""
import pytest
import torch

from gyrodx.engine import Engine

pytestmark = pytest.mark.gpu
ULP = 2.0 ** -24


@pytest.fixture(scope="module")
def eng():
    e = Engine(max_tok=8)
    yield e
    e.close()


def stream():
    return torch.cuda.current_stream().cuda_stream


def test_masked_part_of_a_long_row(eng):
    """A part of a row that holds nothing but 3.6e8 masked logits of the type's lowest value: joined with the other part
    it adds nothing, though its sum times the distance of the maxima is past fp32's range. 512 rows take two parts each;
    they are one row in memory.

    The other part has 1000 logits that count, each within 4 2^-24 (1 + |d|), summed in at most 64 steps."""
    n, V, kept = 512, 720_000_000, 1000
    print(f"{n} rows of {V} logits, {V - kept} masked", flush=True)
    row = torch.full((1, V), torch.finfo(torch.bfloat16).min, dtype=torch.bfloat16, device="cuda")
    x = torch.randn(kept, generator=torch.Generator().manual_seed(3)).bfloat16()
    at = torch.arange(kept) * 13 + V - 20_000
    row[0, at.cuda()] = x.cuda()
    tokens = torch.tensor([[int(at[7]), 5]], device="cuda").expand(n, 2).contiguous()
    lp, H = torch.full((n, 2), 7.0, device="cuda"), torch.full((n,), 7.0, device="cuda")
    ws = torch.empty(eng.logprobs_workspace(n, V), dtype=torch.uint8, device="cuda")
    eng.logprobs(row.expand(n, V), ws, tokens=tokens, logprob=lp, entropy=H, stream=stream())
    torch.cuda.synchronize()
    d = x.double() - x.double().max()
    S, T = d.exp().sum(), (d * d.exp()).sum()
    logs, ts = float(S.log()), float((T / S).abs())
    rel = (64 + 4 * (1 + float(d.abs().max()))) * ULP
    entropy, own = float((H.cpu().double() - (logs + ts)).abs().max()), float((lp[:, 0].cpu().double() - (float(d[7]) - logs)).abs().max())
    assert entropy <= rel * (2 + 2 * ts) + 4 * ULP * (logs + 1)
    assert own <= rel + 4 * ULP * (abs(float(d[7])) + logs + 1)
    assert bool((lp[:, 1] < -3e38).all())


def test_one_workspace_for_every_batch(eng):
    """A workspace taken for 1024 rows serves the smaller batches, which are split over more groups a row; S sums 20000
    terms, each within 4 2^-24 (1 + |d|) and |d| < 25, at most 20000 / 256 + 32 in a row."""
    V, top = 20_000, 5
    ws = torch.full((eng.logprobs_workspace(1024, V, top),), 0xA5, dtype=torch.uint8, device="cuda")
    x = torch.randn(1024, V, generator=torch.Generator().manual_seed(4)) * 2.5
    want = torch.log_softmax(x.double(), -1)
    xd, tol = x.cuda(), (V / 256 + 32 + 4 * 26) * ULP + 8 * ULP * 25
    for n in (1024, 1, 64, 513, 300, 37, 512):
        print(f"{n} rows in the workspace of 1024", flush=True)
        ids, lp = torch.full((n, top), -1, dtype=torch.int32, device="cuda"), torch.zeros(n, top, device="cuda")
        eng.logprobs(xd[:n], ws, top_ids=ids, top_logprobs=lp, stream=stream())
        best = torch.sort(x[:n], dim=-1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(ids.cpu().long(), best)
        assert float((lp.cpu().double() - want[:n].gather(1, best)).abs().max()) <= tol

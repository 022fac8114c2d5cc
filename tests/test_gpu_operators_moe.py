"""The operators around a MoE layer, as a decode step has them: the norm before the layer, the layer, the residual step behind
it, the 4-bit head and the log probabilities, all on device rows and one stream."""
import numpy as np
import pytest
import torch

import op_reference as ref
from gyrodx import synth
from gyrodx.engine import PATH_DECODE, Engine

pytestmark = pytest.mark.gpu
E, V, TOP = 1024, 3001, 7


class Block:
    """A MoE layer with a shared expert between two norms, then the head."""

    def __init__(self, n):
        rng = np.random.default_rng(41)
        self.n, self.layer = n, synth.make_layer(42, E=E, F=512, n_expert=32, n_used=8, mixed_types=True, SF=512)
        self.eng = Engine(max_tok=8)
        self.index = self.eng.add_layer(self.layer)
        data, self.W, _, _ = ref.random_matrix(rng, "q4_1", V, E, 32, True, False)
        self.head = self.eng.add_matrix("q4_1", V, E, data)
        self.eng.load_operators()
        z = lambda *s, t=torch.float32: torch.zeros(*s, device="cuda", dtype=t)  # noqa: E731
        self.x, self.before, self.moe, self.out, self.after = (z(n, E) for _ in range(5))
        self.logits, self.lp, self.H = z(n, V), z(n, 1), z(n)
        self.ids, self.top, self.tokens = z(n, TOP, t=torch.int32), z(n, TOP), z(n, 1, t=torch.int64)
        self.ws = z(max(1, self.eng.logprobs_workspace(n, V, TOP)), t=torch.uint8)
        self.w = [torch.from_numpy(1 + 0.1 * rng.standard_normal(E)).float().cuda() for _ in range(3)]
        self.gate = torch.from_numpy(rng.standard_normal((n, 1))).float().cuda()

    def set(self, seed):
        g = torch.Generator().manual_seed(seed)
        self.x.copy_(torch.randn(self.n, E, generator=g))
        self.tokens.copy_(torch.randint(0, V, (self.n, 1), generator=g))

    def run(self):
        e, s = self.eng, torch.cuda.current_stream().cuda_stream
        e.block_norm(None, self.x, None, self.before, pre_weight=self.w[0], stream=s)
        # (To the layer's call 0 is the engine's compute stream, and 1, hipStreamLegacy, the default stream.)
        e.forward_decode_noalloc(self.index, self.before.data_ptr(), self.n, self.moe.data_ptr(), s or 1)
        e.block_norm(self.moe, self.x, self.out, self.after, post=True, post_weight=self.w[1], gate=self.gate,
                     gate_act="sigmoid", scale=0.5, pre_weight=self.w[2], stream=s)
        e.linear(self.head, self.after, self.logits, stream=s)
        e.logprobs(self.logits, self.ws, tokens=self.tokens, logprob=self.lp, entropy=self.H, top_ids=self.ids,
                   top_logprobs=self.top, stream=s)

    def outputs(self):
        return [t.clone() for t in (self.before, self.moe, self.out, self.after, self.logits, self.lp, self.H, self.ids, self.top)]

    def check(self):
        """The layer equals its own host call bit for bit. Each operator against 64 bits on what it was given: a norm's value
        goes through at most 64 roundings and half of as many in its root; a product adds (76 + groups) roundings of up to 55 / 4.6
        of its size, as often up as down; the log probabilities as far as fp32's sums of 3001 terms."""
        c = lambda t: t.cpu().double()  # noqa: E731
        ulp = 2.0 ** -24
        _, z, _ = ref.block_norm(None, c(self.x), False, None, 0, None, None, 1, c(self.w[0]), 1e-6)
        assert ((c(self.before) - z).abs() <= 64 * ulp * z.abs()).all()
        host = self.eng.forward(self.index, self.before.cpu().numpy(), PATH_DECODE)
        np.testing.assert_array_equal(self.moe.cpu().numpy().view(np.uint32), host.view(np.uint32))
        v, z, part = ref.block_norm(c(self.moe), c(self.x), True, c(self.w[1]), 1e-6, c(self.gate), "sigmoid", 0.5, c(self.w[2]), 1e-6)
        assert part.abs().max() > 0.01 and ((c(self.out) - v).abs() <= 2 * ulp * v.abs() + 64 * ulp * part.abs()).all()
        assert (c(self.after) - z).norm() <= 1e-5 * z.norm()
        y = c(self.after) @ self.W.T
        assert (c(self.logits) - y).norm() <= 12 * np.sqrt(76 + E // 32) * ulp * y.norm()
        lp, H, every, *_ = ref.logprobs(c(self.logits), self.tokens.cpu(), 1.0)
        best = ref.order(self.logits.cpu())[:, :TOP]
        assert torch.equal(self.ids.cpu().long(), best)
        for got, want in ((self.lp, lp), (self.H, H), (self.top, every.gather(1, best))):
            assert ((c(got) - want).abs() <= 1e-5 * (1 + want.abs())).all()


@pytest.mark.parametrize("n", [1, 3, 8])
def test_decode_step(n):
    """Eager on a side stream, then captured and replayed with eager steps on the default stream and host calls of the layer
    between."""
    print(f"MoE layer and operators, {n} tokens", flush=True)
    b, side = Block(n), torch.cuda.Stream()
    try:
        wants = []
        for seed in range(3):
            b.set(seed)
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                b.run()
            side.synchronize()
            b.check()
            wants.append(b.outputs())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            b.run()
        for turn in range(4):
            print(f"replay {turn}", flush=True)
            b.set(turn % 3)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(got, want) for got, want in zip(b.outputs(), wants[turn % 3]))
            b.set((turn + 1) % 3)
            b.run()
            torch.cuda.synchronize()
            b.check()
        del graph
    finally:
        b.eng.close()

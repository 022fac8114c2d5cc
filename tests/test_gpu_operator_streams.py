"""The operators on torch's current stream, which a call without a stream goes to."""
import numpy as np
import pytest
import torch

import op_reference as ref
from gyrodx.engine import Engine

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = Engine(max_tok=8)
    e.load_operators()
    yield e
    e.close()


class Step:
    """A product with a 4-bit matrix, the norm of its rows, their entropy and top, without a stream in any call."""

    def __init__(self, eng):
        rng = np.random.default_rng(31)
        data, self.W, _, _ = ref.random_matrix(rng, "q4_0", 160, 256, 32, False, True)
        self.eng, self.matrix = eng, eng.add_matrix("q4_0", 160, 256, data)
        self.x, self.y, self.normed = (torch.zeros(4, s, device="cuda") for s in (256, 160, 160))
        self.ids, self.top = torch.zeros(4, 3, dtype=torch.int32, device="cuda"), torch.zeros(4, 3, device="cuda")

    def run(self):
        self.eng.linear(self.matrix, self.x, self.y)
        self.eng.block_norm(None, self.y, None, self.normed)
        self.eng.logprobs(self.normed, top_ids=self.ids, top_logprobs=self.top)

    def check(self, xs):
        want = xs.double() @ self.W.T
        assert torch.equal(self.y.cpu().double(), want)
        # A mean of 160 squares and its root: 64 roundings, as for longer rows.
        z = want / torch.sqrt((want * want).mean(-1, keepdim=True) + 1e-6)
        assert ((self.normed.cpu().double() - z).abs() <= 64 * 2.0 ** -24 * z.abs()).all()
        assert torch.equal(self.ids.cpu().long(), ref.order(self.normed.cpu())[:, :3])


def tokens(i):
    return torch.randint(-3, 4, (4, 256), generator=torch.Generator().manual_seed(i)).float()


def test_side_stream(eng):
    """On a side stream the calls follow the work queued there before them."""
    step, side = Step(eng), torch.cuda.Stream()
    busy = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for i in range(4):
        print(f"side stream, step {i}", flush=True)
        xs = tokens(i).cuda()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(4):
                busy = (busy @ busy).clamp_(-1, 1)  # the inputs arrive late
            step.x.copy_(xs)
            step.run()
        side.synchronize()
        step.check(tokens(i))
    eng.release_matrix(step.matrix)


def test_capture(eng):
    """In a capture the calls are recorded; every replay works on the inputs of its time."""
    step = Step(eng)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.run()
    for i in range(4):
        print(f"capture, replay {i}", flush=True)
        step.x.copy_(tokens(10 + i))
        graph.replay()
        torch.cuda.synchronize()
        step.check(tokens(10 + i))
        step.x.copy_(tokens(20 + i))
        step.run()
        torch.cuda.synchronize()
        step.check(tokens(20 + i))
    eng.release_matrix(step.matrix)

"""The operators of a step that checks drafted tokens, one behind the other as a model runs them: queries from 4-bit weights, attention behind
a shared prefix, logits from 4-bit weights, the drafts' test."""
import math

import pytest
import torch

from tests import test_gpu_attention_shared as shared
from tests import test_gpu_gemm_q4 as q4
from tests import test_gpu_verify as verify

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
VOCAB, HIDDEN = 500, 96


class Step:
    """Every part's inputs and outputs stay, so that each is held against the 64-bit form of what it was given."""

    def __init__(self, dtype, seed=0, room=None):
        from sprout_lm_amd import ops
        self.dtype, self.case = dtype, shared.Case(dtype, 4, 2, 32, 16, 100, [(3, 5), (1, 17), (4, 9)], seed=seed, extra_rows=0)
        case = self.case
        case.fill()
        self.T = case.T
        self.wq, self.wl = q4.weights(128, HIDDEN, 32, seed=1), q4.weights(VOCAB, 128, 64, seed=2, scale_dtype=F32)
        self.matrices = [ops.q4_pack(codes.to(DEV), scales.to(DEV), group) for (codes, scales, _), group in ((self.wq, 32), (self.wl, 64))]
        self.k, self.v, self.tables = case.k.to(DEV), case.v.to(DEV), case.tables.to(DEV)
        self.batch = ops.AttentionBatch.build([n for n, _ in case.seqs], [100 + n for _, n in case.seqs], DEV)
        new = lambda *shape, of=dtype: torch.full(shape, 7, dtype=of, device=DEV)
        self.x, self.q, self.o, self.logits = new(self.T, HIDDEN), new(self.T, 128), new(self.T, 128), new(self.T, VOCAB)
        self.tokens, self.uniform = new(self.T, of=torch.int32), new(self.T, of=F32)
        self.starts, self.lens = (torch.tensor(a, dtype=torch.int32, device=DEV) for a in ([0, 3, 4], [3, 1, 4]))
        self.temperature = torch.tensor([0.0, 0.7, 1.1], device=DEV)
        self.accepted, self.following = new(3, of=torch.int32), new(3, of=torch.int32)
        self.workspace = new(ops.verify_workspace_floats(self.T, 3, VOCAB), of=F32)
        self.rooms = {}

    def room(self, name):
        def give(n):
            if name not in self.rooms or self.rooms[name].numel() < n:
                self.rooms[name] = torch.full((n,), math.nan, device=DEV)
            return self.rooms[name]
        return give

    def feed(self, seed):
        g = torch.Generator().manual_seed(seed)
        self.x.copy_(torch.randn(self.T, HIDDEN, generator=g).mul_(0.4))
        self.uniform.copy_(torch.rand(self.T, generator=g))
        self.tokens.copy_(torch.randint(0, VOCAB, (self.T,), generator=g))

    def run(self):
        from sprout_lm_amd import ops
        ops.gemm_q4(self.x, self.matrices[0], self.q, workspace=self.room("q"))
        ops.attention_shared(self.q, 128, self.k, self.v, self.tables, self.batch, 100, self.o, 4, 2, 32, 32 ** -0.5, workspace=self.room("o"))
        ops.gemm_q4(self.o, self.matrices[1], self.logits, workspace=self.room("logits"))
        ops.verify_drafts(self.logits, self.tokens, self.starts, self.lens, self.uniform, self.accepted, self.following, self.workspace, self.temperature)

    def check(self):
        torch.cuda.synchronize()
        x, q, o, logits = (t.cpu() for t in (self.x, self.q, self.o, self.logits))
        for a, (codes, scales, w), group, out in ((x, self.wq, 32, q), (o, self.wl, 64, logits)):
            want = a.double() @ w.t()
            assert ((out.double() - want).abs() <= q4.allowed(a, scales, w, group, self.dtype, want)).all()
        self.case.q = q
        self.case.check(o.double(), *self.case.definition())
        expected = verify.definition(logits, self.tokens.cpu(), [0, 3, 4], [3, 1, 4], self.uniform.cpu(), self.temperature.cpu(), None, None)
        assert (self.accepted.tolist(), self.following.tolist()) == expected
        return expected

    def outputs(self):
        return [t.clone() for t in (self.q, self.o, self.logits, self.accepted, self.following)]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_a_step(dtype):
    step = Step(dtype)
    held = 0
    for seed in range(4):
        step.feed(seed)
        if seed % 2:      # drafts that are likely to hold: what the target says itself
            step.run()
            best = step.logits.argmax(-1).int()
            step.tokens[1:] = best[:-1]
        step.run()
        held += sum(step.check()[0])
    assert held > 0


def test_two_recorded_steps_at_once():
    """Two recorded steps with workspaces of their own, replayed on two streams over each other, and an eager one between."""
    steps = [Step(BF16, seed=s) for s in range(2)]
    graphs, streams = [], [torch.cuda.Stream() for _ in steps]
    for step in steps:
        step.feed(0)
        step.run()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            step.run()
        graphs.append(graph)
    for seed in range(1, 5):
        wanted = []
        for i, step in enumerate(steps):
            step.feed(10 * seed + i)
            step.run()
            wanted.append(step.outputs())
            for t in (step.q, step.o, step.logits, step.accepted, step.following, step.workspace, *step.rooms.values()):
                t.fill_(7)
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for step, want in zip(steps, wanted):
            assert all(torch.equal(a, b) for a, b in zip(step.outputs(), want))
            step.check()


def test_the_sampler_tests_drafts():
    """`Sampler.verify`: the tokens of `ops.verify_drafts` under numbers that depend on seed, counter and place alone."""
    from sprout_lm_amd.sampling import NonFiniteLogits, Sampler, SamplingParams
    from sprout_lm_amd.sampling.sampler import uniform_numbers
    data = verify.inputs(700, [3, 1, 5, 2], seed=4)
    params = [SamplingParams(0.9, seed=11), SamplingParams(0.0), SamplingParams(1.2, seed=12), SamplingParams(0.5, seed=2 ** 62)]
    counters, sampler = [5, 0, 19, 2], Sampler(torch.device(DEV), 700)
    logits, drafters = data["logits"].to(DEV), data["draft_logits"].to(DEV)
    tokens, rows = data["tokens"].int().to(DEV), data["draft_rows"].int().to(DEV)
    got = sampler.verify(logits, tokens, [3, 1, 5, 2], params, counters, drafters, rows)
    uniform = uniform_numbers([p.seed for p in params], counters, [3, 1, 5, 2])
    accepted, following = verify.definition(**{**data, "uniform": uniform}, temperature=torch.tensor([p.temperature for p in params]))
    assert got == [[int(t) for t in data["tokens"][start + 1:start + 1 + n]] + [token] for start, n, token in zip(data["starts"], accepted, following)]
    # one sequence alone, and greedy ones
    assert sampler.verify(logits[4:9], tokens[4:9].contiguous(), [5], params[2:3], counters[2:3], drafters, rows[4:9].contiguous()) == got[2:3]
    greedy = sampler.verify(logits, tokens, [3, 1, 5, 2], [SamplingParams()] * 4, counters)
    assert greedy == [[int(t) for t in data["tokens"][s + 1:s + 1 + a]] + [b] for s, a, b in
                      zip(data["starts"], *verify.definition(**{**data, "draft_logits": None, "draft_rows": None}, temperature=None))]
    assert sampler.verify(logits[:0], tokens[:0], [], [], []) == []
    logits[3] = math.nan
    with pytest.raises(NonFiniteLogits):
        sampler.verify(logits, tokens, [3, 1, 5, 2], params, counters, drafters, rows)

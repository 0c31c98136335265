"""Drafted tokens tested against the target's probabilities: the definition in 64 bits, edges of it, and what it leaves distributed."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def definition(logits, tokens, starts, lens, uniform, temperature, draft_logits, draft_rows):
    accepted, following = [], []
    for s, (start, n) in enumerate(zip(starts, lens)):
        warm = 0.0 if temperature is None else float(temperature[s])
        hold, token = 0, -1
        for j in range(n):
            row = logits[start + j].double()
            hold = j
            if not bool((row < math.inf).all()) or not bool((row > -math.inf).any()):
                break
            if warm <= 0.0:
                token = int((row == row.max()).nonzero()[0])
                if j < n - 1 and int(tokens[start + j + 1]) == token:
                    token = -1
                    continue
                break
            p = torch.softmax(row / warm, 0)
            if j < n - 1:
                draft, q = int(tokens[start + j + 1]), torch.zeros_like(p)
                source = -1 if draft_rows is None else int(draft_rows[start + j + 1])
                known = 0 <= draft < len(p)
                if source >= 0:
                    other = draft_logits[source].double() if source < len(draft_logits) else torch.full_like(row, math.nan)
                    if not bool((other < math.inf).all()) or not bool((other > -math.inf).any()):
                        break
                    q = torch.softmax(other / warm, 0)
                elif known:
                    q[draft] = 1.0
                if known and float(uniform[start + j]) * float(q[draft]) < float(p[draft]):
                    continue
                left = (p - q).clamp_min(0.0)
                p = left if float(left.sum()) > 0 else p
            running = torch.cumsum(p, 0)
            over = running > float(uniform[start + n - 1]) * running[-1]
            token = int(over.nonzero()[0])
            break
        accepted.append(hold)
        following.append(token)
    return accepted, following


def call(logits, tokens, starts, lens, uniform, temperature=None, draft_logits=None, draft_rows=None):
    from sprout_lm_amd import ops
    to = lambda t: None if t is None else t.to(DEV).contiguous()
    ints = lambda a: torch.as_tensor(a, dtype=torch.int32).to(DEV)
    n = len(starts)
    accepted, following = (torch.full((n + 1,), 77, dtype=torch.int32, device=DEV) for _ in range(2))
    workspace = torch.full((ops.verify_workspace_floats(*([logits.shape[0], n, logits.shape[1]])),), math.nan, device=DEV)
    ops.verify_drafts(to(logits), ints(tokens), ints(starts), ints(lens), to(uniform), accepted, following, workspace, to(temperature), to(draft_logits),
                      None if draft_rows is None else ints(draft_rows))
    assert accepted[n] == 77 and following[n] == 77
    return accepted[:n].tolist(), following[:n].tolist()


def inputs(vocab, lens, seed, drawn=1.0, dtype=torch.float32, gap=0):
    """Rows of sequences of `lens` rows, `gap` unused rows between them; a share `drawn` of the drafts from a drafter's row, the others guessed."""
    g = torch.Generator().manual_seed(seed)
    starts, at = [], 0
    for n in lens:
        starts.append(at)
        at += n + gap
    logits = torch.randn(at, vocab, generator=g).mul_(2.5).to(dtype)
    tokens, rows, drafters = torch.randint(0, vocab, (at,), generator=g), torch.full((at,), -1), []
    for start, n in zip(starts, lens):
        for j in range(n - 1):
            if torch.rand((), generator=g) < drawn:
                other = (logits[start + j].float() + 0.5 * torch.randn(vocab, generator=g)).to(dtype)
                rows[start + j + 1] = len(drafters)
                drafters.append(other)
                tokens[start + j + 1] = torch.multinomial(torch.softmax(other.float(), 0), 1, generator=g)[0]
            elif torch.rand((), generator=g) < 0.6:
                tokens[start + j + 1] = logits[start + j].float().argmax()
    drafters = torch.stack(drafters) if drafters else torch.zeros(1, vocab, dtype=dtype)
    return dict(logits=logits, tokens=tokens, starts=starts, lens=list(lens), uniform=torch.rand(at, generator=g), draft_logits=drafters, draft_rows=rows)


def check(data):
    got, want = call(**data), definition(**data)
    assert got[0] == want[0] and got[1] == want[1]
    return got


@pytest.mark.parametrize("vocab", [1, 2, 5, 63, 1000, 4095, 4096, 4097, 32771, 151936])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_against_the_definition(vocab, dtype):
    lens = [1, 2, 5, 8, 3, 1, 12] if vocab < 100000 else [1, 5, 3]
    data = inputs(vocab, lens, seed=vocab, drawn=0.7, dtype=dtype, gap=vocab % 2)
    for warmth in (1.0, 0.7):
        check(dict(data, temperature=torch.full((len(lens),), warmth)))
    mixed = torch.tensor([0.0, 1.0, 0.0, 1.7, 0.3, 0.0, 0.9])[:len(lens)]
    check(dict(data, temperature=mixed))
    check(dict(data, temperature=None, uniform=None))
    check(dict(data, temperature=mixed, draft_logits=None, draft_rows=None))


@pytest.mark.parametrize("sequences", [1, 64, 257, 700])
def test_many_sequences(sequences):
    lens = [1 + i % 7 for i in range(sequences)]
    got = check(dict(inputs(503, lens, seed=sequences), temperature=torch.ones(sequences)))
    assert sequences == 1 or (0 < sum(got[0]) < sum(lens) - sequences)      # some drafts hold, some do not


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("vocab", [17000, 17001])
def test_many_sequences_of_many_chunks(vocab, dtype):
    """So many that decisions are a launch of their own; among them rows that are not there and rows of two sequences."""
    lens = [1 + i % 5 for i in range(160)]
    data = inputs(vocab, lens, seed=vocab, dtype=dtype)
    temperature = torch.tensor([0.0, 1.0, 0.6, 1.3])[torch.arange(160) % 4]
    check(dict(data, temperature=temperature))
    rows = len(data["logits"])
    more = {**data, "starts": data["starts"] + [rows - 1, -4, data["starts"][7]], "lens": lens + [2, 3, 1]}      # the last: the eighth sequence's first row
    accepted, following = call(**more, temperature=torch.cat([temperature, torch.ones(3)]))
    wanted = definition(**data, temperature=temperature)
    keep = [i for i in range(160) if i != 7]
    assert [accepted[i] for i in keep] == [wanted[0][i] for i in keep] and [following[i] for i in keep] == [wanted[1][i] for i in keep]
    assert accepted[160:] == [0, 0, 0] and following[160:] == [-1, -1, -1] and (accepted[7], following[7]) == (0, -1)


def test_numbers_at_their_ends():
    """The smallest and the largest uniform number; tokens that are not allowed before and behind the only one that is."""
    data = inputs(300, [3, 3, 3, 3], seed=5)
    data["logits"][:, :100], data["logits"][:, 200:] = -math.inf, -math.inf
    for u in (0.0, 1.0 - 2.0 ** -24):
        got = check(dict(data, temperature=torch.ones(4), uniform=torch.full((12,), u)))
        assert all(100 <= t < 200 for t in got[1])
    data["logits"][:] = -math.inf
    data["logits"][:, 299] = -3.0e38
    got = check(dict(data, temperature=torch.full((4,), 0.01)))
    assert got[1] == [299] * 4


def test_equal_rows_hold_every_draft():
    data = inputs(1000, [6, 6], seed=3)
    for s in data["starts"]:
        for j in range(5):
            data["draft_logits"][data["draft_rows"][s + j + 1]] = data["logits"][s + j]
    data["uniform"][:] = 1.0 - 2.0 ** -24
    assert check(dict(data, temperature=torch.ones(2)))[0] == [5, 5]


def test_a_draft_that_neither_side_allows():
    """p(draft) = q(draft) = 0 under equal rows: nothing is left of p - q, the next token comes from p."""
    data = inputs(5000, [2], seed=3)
    data["logits"][0, 17] = -math.inf
    data["draft_logits"][0] = data["logits"][0]
    data["tokens"][1] = 17
    assert check(dict(data, temperature=torch.ones(1)))[0] == [0]


def test_ties_go_to_the_lowest_index():
    data = inputs(9000, [3, 2], seed=8)
    data["logits"][:] = 0.0
    data["logits"][:, 7000], data["logits"][:, 4097], data["logits"][1, 12] = 1.0, 1.0, 1.0
    data["tokens"][:] = 4097
    assert check(dict(data, temperature=None)) == ([1, 1], [12, 4097])


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("warmth", [0.0, 1.0])
def test_rows_that_are_not_finite(bad, warmth):
    """The deciding row gives -1; a row behind it does not matter."""
    data = inputs(5000, [4, 4, 4, 4, 1], seed=1)
    for s in range(4):      # every draft holds
        for j in range(3):
            at = data["starts"][s] + j
            data["tokens"][at + 1] = data["logits"][at].argmax()
    data["uniform"][:] = 0.0
    data["logits"][0 + 1, 4999] = bad                       # the second row of the first sequence
    data["logits"][4 + 3, 3] = bad                          # the last of the second
    data["logits"][12 + 2] = -math.inf
    data["tokens"][12 + 1] = (int(data["tokens"][12 + 1]) + 1) % 5000      # the fourth, greedy: its first draft fails before the bad row
    if warmth:
        data["uniform"][12] = 0.999999
        data["draft_logits"][data["draft_rows"][8 + 2], 5] = bad      # the third sequence: the second draft's own row
    data["logits"][16] = -math.inf
    got = check(dict(data, temperature=torch.full((5,), warmth)))
    assert got[0][:2] == [1, 3] and got[1][:2] == [-1, -1] and got[1][4] == -1 and (warmth or got[1][3] >= 0)


def test_ids_and_rows_out_of_range():
    data = inputs(700, [3, 3, 3], seed=4)
    data["tokens"][1], data["tokens"][4] = 700, -1            # no tokens of this vocabulary: do not hold
    data["draft_rows"][7] = 1000                              # no row of the drafter's: as a row that is not finite
    got = check(dict(data, temperature=torch.ones(3)))
    assert got[0] == [0, 0, 0] and got[1][2] == -1 and min(got[1][:2]) >= 0
    data["starts"], data["lens"] = [0, -1, 7], [0, 3, 3]      # sequences without rows, or with rows that are not there
    assert call(**dict(data, temperature=torch.ones(3))) == ([0, 0, 0], [-1, -1, -1])


def test_tokens_are_distributed_as_the_target_has_them():
    """The first token of 8,000 sequences with one draft each: counts within five standard deviations of p."""
    n, vocab = 8000, 6
    g = torch.Generator().manual_seed(0)
    p_row, q_row = torch.randn(vocab, generator=g) * 1.5, torch.randn(vocab, generator=g) * 1.5
    q = torch.softmax(q_row / 0.8, 0)
    drafts = torch.multinomial(q, n, replacement=True, generator=g)
    tokens = torch.zeros(2 * n, dtype=torch.long)
    tokens[1::2] = drafts
    rows = torch.zeros(2 * n, dtype=torch.long)
    accepted, following = call(p_row.expand(2 * n, vocab), tokens, list(range(0, 2 * n, 2)), [2] * n, torch.rand(2 * n, generator=g),
                               torch.full((n,), 0.8), q_row[None], rows)
    first = [int(d) if a else t for a, t, d in zip(accepted, following, drafts)]
    p = torch.softmax(p_row.double() / 0.8, 0)
    for token in range(vocab):
        expected = n * float(p[token])
        assert abs(first.count(token) - expected) <= 5 * math.sqrt(expected * (1 - float(p[token]))) + 1, token
    assert 0.05 * n < sum(accepted) < 0.95 * n


def test_from_a_graph_and_on_another_stream():
    from sprout_lm_amd import ops
    data = inputs(20000, [4, 2, 1, 6], seed=9)
    dev = {k: (v.to(DEV).contiguous() if isinstance(v, torch.Tensor) else torch.tensor(v, dtype=torch.int32, device=DEV)) for k, v in data.items()}
    dev["tokens"], dev["draft_rows"] = dev["tokens"].int(), dev["draft_rows"].int()
    temperature = torch.ones(4, device=DEV)
    workspace = torch.empty(ops.verify_workspace_floats(len(data["logits"]), 4, 20000), device=DEV)
    accepted, following = torch.zeros(4, dtype=torch.int32, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV)
    run = lambda: ops.verify_drafts(dev["logits"], dev["tokens"], dev["starts"], dev["lens"], dev["uniform"], accepted, following, workspace, temperature,
                                    dev["draft_logits"], dev["draft_rows"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    assert (accepted.tolist(), following.tolist()) == definition(**data, temperature=torch.ones(4))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for seed in range(4):
        data["uniform"] = torch.rand(len(data["uniform"]), generator=torch.Generator().manual_seed(seed))
        dev["uniform"].copy_(data["uniform"])
        workspace.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert (accepted.tolist(), following.tolist()) == definition(**data, temperature=torch.ones(4))


@pytest.mark.parametrize("warmth", [None, 1.0], ids=["greedy", "drawn"])
def test_rows_of_two_sequences(warmth):
    """A row has one temperature: sequences that share rows are not answered, their neighbours are, also beside ranges that are not there."""
    data = inputs(300, [2, 3, 1, 2], seed=6)
    temperature = None if warmth is None else torch.full((4,), warmth)
    accepted, following = call(**data, temperature=temperature)
    wanted = definition(**data, temperature=temperature)
    assert (accepted, following) == wanted
    more = None if warmth is None else torch.full((8,), warmth)
    rows = {**data, "starts": data["starts"] + [3, -1, 7, 4], "lens": data["lens"] + [2, 9, 2, 0]}      # rows 3 and 4 of the second; -1 ..; 7 and 8; none
    accepted, following = call(**rows, temperature=more)
    assert accepted == [wanted[0][0], 0, wanted[0][2], wanted[0][3], 0, 0, 0, 0]
    assert following == [wanted[1][0], -1, wanted[1][2], wanted[1][3], -1, -1, -1, -1]


@pytest.mark.parametrize("warmth", [-1.0, math.nan])
def test_temperatures_below_zero_are_greedy(warmth):
    data = inputs(300, [2, 3], seed=12)
    assert call(**data, temperature=torch.tensor([warmth, 1.0])) == definition(**data, temperature=torch.tensor([0.0, 1.0]))


def test_a_drafter_without_rows():
    data = inputs(90, [3, 2], seed=8, drawn=0.0)
    data["draft_logits"] = torch.zeros(0, 90)
    assert call(**data, temperature=torch.ones(2)) == definition(**data, temperature=torch.ones(2))


@pytest.mark.parametrize("what", ["dtype", "ints", "uniform", "missing", "pair", "draft", "workspace", "cpu", "rows"])
def test_refusals(what):
    from sprout_lm_amd import ops
    ints = lambda n: torch.ones(n, dtype=torch.int32, device=DEV)
    args = dict(logits=torch.zeros(4, 50, device=DEV), tokens=ints(4), starts=ints(2) * 0, lens=ints(2), uniform=torch.zeros(4, device=DEV), accepted=ints(2),
                next_token=ints(2), workspace=torch.zeros(ops.verify_workspace_floats(4, 2, 50), device=DEV), temperature=torch.ones(2, device=DEV),
                draft_logits=torch.zeros(3, 50, device=DEV), draft_rows=ints(4))
    ops.verify_drafts(**args)
    changed = {"dtype": dict(logits=args["logits"].half(), draft_logits=args["draft_logits"].half()), "ints": dict(tokens=ints(4).long()),
               "uniform": dict(uniform=torch.zeros(3, device=DEV)), "missing": dict(uniform=None), "pair": dict(draft_rows=None),
               "draft": dict(draft_logits=torch.zeros(3, 49, device=DEV)), "workspace": dict(workspace=args["workspace"][:-2].contiguous()),
               "cpu": dict(tokens=ints(4).cpu()), "rows": dict(draft_rows=ints(3))}[what]
    with pytest.raises(ops.KernelError):
        ops.verify_drafts(**{**args, **changed})

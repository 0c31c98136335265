"""Attention behind a shared prefix against the definition in 64 bits, sequence by sequence and head by head."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


class Case:
    """Pools whose free slots hold NaN, block tables that begin with the same pages, queries.  seqs: (queries, own keys)."""

    def __init__(self, dtype, nq, nkv, hd, page, prefix, seqs, seed=0, extra_rows=2, pool=0):
        self.nq, self.nkv, self.hd, self.page, self.prefix, self.seqs, self.dtype = nq, nkv, hd, page, prefix, seqs, dtype
        g = torch.Generator().manual_seed(seed)
        whole = prefix // page
        own = [-(-(prefix + n) // page) - whole for _, n in seqs]
        total = whole + sum(own)
        order = torch.randperm(total, generator=g)
        self.tables = torch.full((len(seqs), whole + max(own) + 1), -1, dtype=torch.int32)
        at = whole
        for i, n in enumerate(own):
            self.tables[i, :whole] = order[:whole]
            self.tables[i, whole:whole + n] = order[at:at + n]
            at += n
        self.k, self.v = (torch.full(shape, math.nan, dtype=dtype) for shape in ((total, nkv, page, hd), (total, nkv, hd, page)))
        shared = [torch.randn(prefix, nkv, hd, generator=g).mul_(1.3).to(dtype) for _ in range(2)]
        self.keys, self.values = [], []
        for i, (_, n) in enumerate(seqs):
            mine = [torch.randn(n, nkv, hd, generator=g).mul_(1.3).to(dtype) for _ in range(2)]
            self.keys.append(torch.cat([shared[0], mine[0]]))
            self.values.append(torch.cat([shared[1], mine[1]]))
        self.T = sum(q for q, _ in seqs)
        self.q = torch.randn(self.T + extra_rows, nq * hd, generator=g).to(dtype)
        self.offset = max(0, pool - total)      # the used pages lie at the pool's end

    def fill(self):
        for i, (_, n) in enumerate(self.seqs):
            for pos in range(self.prefix + n):
                page = int(self.tables[i, pos // self.page])
                self.k[page, :, pos % self.page] = self.keys[i][pos]
                self.v[page, :, :, pos % self.page] = self.values[i][pos]

    def run(self, **options):
        from sprout_lm_amd import ops
        self.fill()
        k, v = self.k.to(DEV), self.v.to(DEV)
        tables = self.tables.to(DEV)
        if self.offset:
            big = lambda t: torch.empty(self.offset + t.shape[0], *t.shape[1:], dtype=t.dtype, device=DEV)
            whole_k, whole_v = big(k), big(v)
            whole_k[self.offset:], whole_v[self.offset:] = k, v
            k, v, tables = whole_k, whole_v, torch.where(tables < 0, tables, tables + self.offset)
        out = torch.full((len(self.q), self.nq * self.hd), 7.0, dtype=self.dtype, device=DEV)
        batch = ops.AttentionBatch.build([q for q, _ in self.seqs], [self.prefix + n for _, n in self.seqs], DEV)
        self.call = lambda target=out, **more: ops.attention_shared(self.q_dev, self.nq * self.hd, k, v, tables, batch, self.prefix, target, self.nq,
                                                                    self.nkv, self.hd, self.hd ** -0.5, **{**options, **more})
        self.q_dev = self.q.to(DEV)
        self.call()
        torch.cuda.synchronize()
        assert (out[self.T:] == 7).all()      # rows behind the last sequence stay as they are
        self.out = out
        return out[:self.T].double().cpu()

    def definition(self, cap=0.0, sinks=None):
        """(result, sum of weights times |values|, largest scale sum |q||k|) in float64."""
        G, at, rows, sizes, reach = self.nq // self.nkv, 0, [], [], 0.0
        for (n_q, n), keys, values in zip(self.seqs, self.keys, self.values):
            ctx = self.prefix + n
            for j in range(n_q):
                seen = ctx - n_q + j + 1
                q = self.q[at + j].double().view(self.nkv, G, self.hd)
                k, v = keys[:seen].double(), values[:seen].double()
                s = torch.einsum("hgd,khd->hgk", q, k) * self.hd ** -0.5
                reach = max(reach, float((torch.einsum("hgd,khd->hgk", q.abs(), k.abs()) * self.hd ** -0.5).nan_to_num(0, 0, 0).max()))
                if cap:
                    s = cap * torch.tanh(s / cap)
                top = s.amax(-1, keepdim=True)
                if sinks is not None:
                    sink = sinks.double().view(self.nkv, G, 1)
                    top = torch.maximum(top, sink)
                w = torch.exp(s - top)
                total = w.sum(-1, keepdim=True)
                if sinks is not None:
                    total = total + torch.exp(sink - top)
                rows.append(torch.einsum("hgk,khd->hgd", w / total, v).reshape(-1))
                sizes.append(torch.einsum("hgk,khd->hgd", w / total, v.abs()).reshape(-1))
            at += n_q
        return torch.stack(rows), torch.stack(sizes), reach

    def check(self, got, want, size, reach):
        """A score is a float32 sum of hd products (hd + 4 roundings with the scale's and the maximum's, each 2^-24 of sum |q||k| at most), which
        moves a weight by that times 2 with the exponential's own (2^-22); sums over n keys and the parts' joins are n + 64 roundings; weights are
        rounded to bfloat16 for the product (2^-8) there, and the result to its type (2^-8 or 2^-24)."""
        keys = self.prefix + max(n for _, n in self.seqs)
        weights = 2.0 ** -24 * (2 * (self.hd + 4) * reach * 2 + 8 + keys + 64)
        if self.dtype == BF16:
            weights += 2.0 ** -8
        tolerance = 2 * weights * size + (2.0 ** -8 if self.dtype == BF16 else 2.0 ** -24) * want.abs() + 1e-30
        off = (got - want).abs()
        assert (off <= tolerance).all(), f"off by {float((off / tolerance).max()):.2f} times what roundings allow"


def check(case, **options):
    got = case.run(**{k: v for k, v in options.items() if k != "definition"})
    case.check(got, *case.definition(**options.get("definition", {})))


# heads, groups, head size, page, prefix, (queries, own keys) of every sequence
CASES = [(4, 2, 64, 16, 100, [(1, 1), (1, 30), (3, 3), (1, 17)]),             # prefix and own keys end inside pages
         (14, 2, 64, 16, 512, [(1, 5)]), (28, 4, 128, 16, 129, [(5, 9), (4, 40), (1, 1)]),
         (3, 1, 64, 16, 0, [(1, 1), (2, 20)]), (3, 3, 32, 8, 1, [(1, 1), (1, 9)]),   # nothing shared, one token shared
         (7, 1, 128, 32, 640, [(40, 45), (1, 2)]),                             # more queries than a tile, more rows than a block
         (24, 2, 64, 16, 77, [(16, 16), (2, 600)]),                            # groups of 12 heads; own keys in two parts
         (2, 1, 96, 16, 200, [(1, 3), (1, 3)]), (5, 5, 48, 16, 70, [(2, 8), (1, 1)]), (2, 2, 192, 16, 150, [(3, 7)]), (4, 1, 256, 16, 90, [(2, 50)]),
         (2, 1, 33, 7, 40, [(2, 5), (1, 1)]), (4, 2, 64, 4, 50, [(1, 6), (3, 3)]), (1, 1, 1, 3, 10, [(1, 4)]), (3, 1, 20, 16, 30, [(1, 9)]),   # sizes no 16-byte piece fits
         (4, 4, 64, 16, 260, [(0, 5), (2, 4), (0, 1), (1, 1)]),                # sequences without queries
         (2, 1, 64, 1, 30, [(1, 3)]), (2, 1, 64, 16, 2300, [(1, 520)] * 3)]


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_against_the_definition(case, dtype):
    check(Case(dtype, *CASES[case], seed=case))


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_own_keys_longer_than_the_shared(dtype):
    check(Case(dtype, 3, 1, 64, 16, 40, [(1, 9000), (2, 4200), (1, 1)], seed=5))


@pytest.mark.parametrize("sequences", [31, 64, 150])
def test_many_sequences(sequences):
    check(Case(BF16, 14, 2, 64, 16, 300, [(1 + i % 3, 3 + i % 29) for i in range(sequences)], seed=sequences))


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_sinks_and_capped_scores(dtype):
    sinks = torch.tensor([2.0, -30.0, 9.0, 0.0])
    check(Case(dtype, 4, 2, 64, 16, 140, [(1, 20), (3, 5)]), sinks=sinks.to(DEV), definition={"sinks": sinks})
    check(Case(dtype, 4, 2, 64, 16, 140, [(1, 20), (3, 5)]), scores="capped", softcap=3.0, definition={"cap": 3.0})


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_a_value_that_is_not_finite_stays_with_the_rows_that_see_its_key(dtype):
    """Drafted tokens behind a query hold NaN and infinities: the query does not see their keys."""
    case = Case(dtype, 4, 2, 64, 16, 100, [(4, 9), (1, 3)])
    case.keys[0][107, 0] = math.nan                         # the third query's own key: seen by it and the fourth
    case.values[0][108, 1, 5] = math.nan                    # the fourth's values
    case.values[0][106, 1, 7], case.values[0][107, 1, 7] = math.inf, -math.inf      # the second's and the third's
    got = case.run().view(5, 2, 2, 64)
    want, size, reach = case.definition()
    want, size = want.view(5, 2, 2, 64), size.view(5, 2, 2, 64)
    assert got[2:4, 0].isnan().all() and torch.equal(got[:, 1].isnan(), want[:, 1].isnan()) and got[3, 1, :, 5].isnan().all()
    assert (got[1, 1, :, 7] == math.inf).all() and got[2, 1, :, 7].isnan().all()
    fine = want.isfinite()
    assert fine[0].all() and fine[4].all() and got[fine].isfinite().all()
    case.check(got[fine], want[fine], size[fine], reach)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_keys_of_no_weight(dtype):
    """Scores of minus infinity weigh nothing, shared and own; scores far apart."""
    case = Case(dtype, 2, 1, 64, 16, 300, [(1, 3), (2, 4)])
    case.q[:, 3], case.q[:, 67] = 1.0, 1.0
    for keys in case.keys:
        keys[5, 0, 3] = -math.inf
        keys[200:, 0, 9] *= 30
    case.keys[0][301, 0, 3] = -math.inf
    got = case.run()
    want, size, _ = case.definition()
    case.check(got, want, size, 300.0)


def test_a_prefix_table_of_its_own():
    case = Case(BF16, 4, 2, 64, 16, 100, [(1, 4), (2, 9)])
    table = case.tables[0, :7].clone().to(DEV)
    case.tables[:, :6] = -1                     # the sequences' own rows do not know the shared pages
    own = case.tables.clone()
    case.tables[:, :6] = table[:6].cpu()        # (for `fill`)
    case.fill()
    case.fill, case.tables = lambda: None, own
    got = case.run(prefix_table=table)
    case.check(got, *case.definition())


def test_offsets_beyond_32_bits():
    """Pools of more than 2^32 bytes and 2^31 numbers whose last pages are used."""
    pages = 2 ** 31 // (2 * 128 * 64) + 40
    check(Case(BF16, 4, 2, 128, 64, 200, [(1, 4), (2, 70)], pool=pages))


def test_page_numbers_outside_the_pool_are_not_followed():
    from sprout_lm_amd import ops
    case = Case(BF16, 4, 2, 64, 16, 100, [(1, 4)])
    case.run()
    bad = torch.full((1, 8), 2 ** 30, dtype=torch.int32, device=DEV)
    bad[0, ::2] = -5
    k, v = case.k.nan_to_num(0).to(DEV), case.v.nan_to_num(0).to(DEV)
    batch = ops.AttentionBatch.build([1], [104], DEV)
    out = torch.zeros(1, 256, dtype=BF16, device=DEV)
    ops.attention_shared(case.q_dev, 256, k, v, bad, batch, 100, out, 4, 2, 64, 0.125)
    torch.cuda.synchronize()


def test_repeats_bit_for_bit_on_another_stream_and_from_a_graph():
    case = Case(BF16, 14, 2, 64, 16, 700, [(1, 40), (3, 700), (2, 9)])
    case.run()
    first = case.out.clone()
    kept = {}

    def workspace(n):
        if "t" not in kept:
            kept["t"] = torch.full((n,), math.nan, device=DEV)      # whatever lay there before does not matter
        return kept["t"]
    side, other = torch.cuda.Stream(), torch.zeros_like(first)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        case.call(other, workspace=workspace)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other[:case.T], first[:case.T])
    graph, target = torch.cuda.CUDAGraph(), torch.zeros_like(first)
    with torch.cuda.graph(graph):
        case.call(target, workspace=workspace)
    queries = case.q_dev.clone()
    for i in range(3):
        case.q_dev.copy_(queries * (1 + i))
        target.zero_()
        graph.replay()
        torch.cuda.synchronize()
        case.call(other)
        assert torch.equal(target[:case.T], other[:case.T])
        kept["t"].fill_(math.nan)


def test_as_the_attention_of_whole_contexts():
    """The same step through `attention`, which reads the prefix once a sequence."""
    from sprout_lm_amd import ops
    case = Case(BF16, 14, 2, 64, 16, 512, [(1, 40), (1, 300), (4, 9)])
    got = case.run()
    k, v = case.k.to(DEV), case.v.to(DEV)
    batch = ops.AttentionBatch.build([q for q, _ in case.seqs], [512 + n for _, n in case.seqs], DEV)
    out = torch.empty(case.T, 14 * 64, dtype=BF16, device=DEV)
    ops.attention(case.q_dev[:case.T].contiguous(), 14 * 64, k.nan_to_num(0), v.nan_to_num(0), case.tables.to(DEV), batch, out, 14, 2, 64, None, 0.125)
    _, size, _ = case.definition()
    # both round weights (2^-8 of each weighted value) and results (2^-8)
    assert ((got - out.double().cpu()).abs() <= 2 * (2.0 ** -8 + 2.0 ** -12) * size + 2 * 2.0 ** -8 * got.abs() + 1e-6).all()


@pytest.mark.parametrize("what", ["prefix", "unknown", "long", "dtype", "head", "stride", "sinks", "table", "workspace", "cpu", "cap"])
def test_refusals(what):
    from sprout_lm_amd import ops
    q = torch.zeros(2, 256, dtype=BF16, device=DEV)
    k, v = torch.zeros(9, 2, 16, 64, dtype=BF16, device=DEV), torch.zeros(9, 2, 64, 16, dtype=BF16, device=DEV)
    tables = torch.zeros(2, 9, dtype=torch.int32, device=DEV)
    batch = ops.AttentionBatch.build([1, 1], [101, 110], DEV)
    args = dict(q=q, q_stride=256, k_pool=k, v_pool=v, block_tables=tables, batch=batch, prefix=100, out=torch.zeros_like(q), nq=4, nkv=2, hd=64, scale=0.125)
    ops.attention_shared(**args)
    changed = {"prefix": dict(prefix=101), "unknown": dict(batch=ops.AttentionBatch(batch.q_start, batch.q_len, batch.ctx_len, 2, batch.lists, 110, 110)),
               "long": dict(batch=ops.AttentionBatch.build([1, 1], [101, 145], DEV)), "dtype": dict(q=q.half(), out=q.half()),
               "head": dict(nq=1, nkv=1, hd=257, k_pool=torch.zeros(9, 1, 16, 257, device=DEV), v_pool=torch.zeros(9, 1, 257, 16, device=DEV)),
               "stride": dict(q_stride=128), "sinks": dict(sinks=torch.zeros(3, device=DEV)),
               "table": dict(prefix_table=torch.zeros(6, dtype=torch.int32, device=DEV)), "workspace": dict(workspace=lambda n: torch.zeros(n - 1, device=DEV)),
               "cpu": dict(block_tables=tables.cpu()), "cap": dict(scores="capped")}[what]
    with pytest.raises(ops.KernelError):
        ops.attention_shared(**{**args, **changed})

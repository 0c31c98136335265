"""The operators of a step that checks drafted tokens for many answers to one prompt, measured one by one.

* `shared`: attention of a batch whose sequences all begin with the same `prefix` tokens, in the paged cache; every sequence brings
  1 to `queries` queries behind its own `own_low` .. `own_high` keys (its queries counted).
* `verify`: drafted tokens tested against the target's probabilities with given random numbers, the next token drawn.
* `q4`: a product with weights of 4 bits and a scale per group of `group` numbers of K.

A case is a dict of plain values; sizes are those of the command line's presets or lie near them.  `prepare` makes the inputs
and what a program keeps between calls, `run` makes one call.  With `own` false the operators are computed in elementary torch operations.
"""
from __future__ import annotations

import math

import torch

own = False

PAGE = 16      # tokens in a page of the cache


# ---------------------------------------------------------------------------------------------- the cases
def _shared(dtype, heads, kv_heads, dim, sequences, queries, prefix, own_low, own_high):
    return {"op": "shared", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "sequences": sequences,
            "queries": queries, "prefix": prefix, "own_low": own_low, "own_high": own_high}


def _verify(vocab, sequences, drafts, temperature, drafter):
    return {"op": "verify", "vocab": vocab, "sequences": sequences, "drafts": drafts, "temperature": temperature, "drafter": drafter}


def _q4(dtype, tokens, rows, cols, group):
    return {"op": "q4", "dtype": dtype, "tokens": tokens, "rows": rows, "cols": cols, "group": group}


def listed() -> list[dict]:
    cases = {
        # four answers to one short question, smallest model: launches and latency
        "shared 0.5b 4x1 behind 500": _shared("bfloat16", 14, 2, 64, 4, 1, 500, 16, 64),
        # a system prompt of ordinary length before 33 conversations, no two equally long
        "shared 7b 33x1 behind 4093": _shared("bfloat16", 28, 4, 128, 33, 1, 4093, 1, 512),
        # the step that checks up to four drafted tokens of each of 64 answers about a document
        "shared 7b 64x5 behind 8192": _shared("bfloat16", 28, 4, 128, 64, 5, 8192, 64, 1024),
        # a document as long as the model reads, 16 questions about it
        "shared 32b 16x1 behind 32000": _shared("bfloat16", 40, 8, 128, 16, 1, 32000, 32, 700),
        # the exact path: float32 numbers throughout
        "shared 0.5b float32 8x3 behind 1500": _shared("float32", 14, 2, 64, 8, 3, 1500, 8, 200),
        # one user's answer with four drafted tokens
        "verify 0.5b 1x4": _verify(151936, 1, 4, 0.8, True),
        # a full server, 1 to 7 drafted tokens an answer
        "verify 7b 64x7": _verify(152064, 64, 7, 1.0, True),
        # drafts looked up in the text, answers without sampling, a vocabulary of an odd size
        "verify greedy 17x3": _verify(32771, 17, 3, 0.0, False),
        # one token through the smallest model's widest reduction
        "q4 0.5b down 1": _q4("bfloat16", 1, 896, 4864, 128),
        # one token, ordinary model: the product that a decoded token spends most of its time in
        "q4 7b gate/up 1": _q4("bfloat16", 1, 37888, 3584, 128),
        # eight answers with four drafted tokens each, on the float32 path
        "q4 7b down 40 float32": _q4("float32", 40, 3584, 18944, 64),
        # a full batch through the largest model, the finest groups
        "q4 32b gate/up 64": _q4("bfloat16", 64, 55296, 5120, 32),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1)) - 0.5 / high))))


def draw(rng) -> dict:
    """Another case of the same ranges: 1 to 64 sequences of 1 to 5 queries behind 16 to 32,000 shared and up to 1,024 own keys;
    1 to 64 answers with 1 to 7 drafts over 1,000 to 152,064 tokens; 1 to 64 tokens by matrices of 100 to 55,296 rows.  None that
    reads or computes more than the largest listed one of its operator."""
    op = rng.choice(["shared", "verify", "q4"])
    most = [work(case) for case in listed() if case["op"] == op]
    while True:
        case = {"shared": _draw_shared, "verify": _draw_verify, "q4": _draw_q4}[op](rng)
        if all(work(case)[what] <= max(w[what] for w in most) for what in ("bytes", "flops")):
            return case


def _draw_shared(rng):
    heads, kv_heads, dim = rng.choice([(14, 2, 64), (28, 4, 128), (40, 8, 128), (16, 2, 64), (5, 5, 48), (32, 4, 128), (3, 1, 32)])
    dtype, queries = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"]), rng.choice([1, 1, 2, 3, 4, 5])
    high = _log_int(rng, queries, 1024)
    return _shared(dtype, heads, kv_heads, dim, _log_int(rng, 1, 64), queries, _log_int(rng, 16, 32000 if dtype == "bfloat16" else 4096),
                   _log_int(rng, 1, high), high)


def _draw_verify(rng):
    return _verify(rng.choice([151936, 152064, 32768, _log_int(rng, 1000, 152064)]), _log_int(rng, 1, 64), rng.randint(1, 7),
                   rng.choice([0.0, 0.6, 0.8, 1.0, 1.3]), rng.random() < 0.7)


def _draw_q4(rng):
    group = rng.choice([32, 64, 128])
    return _q4(rng.choice(["bfloat16", "bfloat16", "float32"]), _log_int(rng, 1, 64), _log_int(rng, 100, 55296),
               group * _log_int(rng, 2, 5120 // group), group)


def _spread(n, low, high):
    return [high] if n == 1 else [round(low * (high / low) ** (i / (n - 1))) for i in range(n)]


def _lengths(case):
    """(queries, own keys) of every sequence: the queries 1 .. `queries` in turn, the keys spread over the logarithm."""
    own_keys = _spread(case["sequences"], case["own_low"], case["own_high"])
    queries = [case["queries"] - i % case["queries"] for i in range(case["sequences"])]
    return [(q, max(q, n)) for q, n in zip(queries, own_keys)]


def _drafts(case):
    """Drafted tokens of every sequence."""
    return [case["drafts"] - i % case["drafts"] for i in range(case["sequences"])]


# ---------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _shared_inputs(case, seed):
    """Pools, block tables whose rows begin with the same pages, queries; scores of a deviation of about 1.7."""
    g, dtype = _generator(seed), getattr(torch, case["dtype"])
    lengths, P, nkv, d = _lengths(case), case["prefix"], case["kv_heads"], case["dim"]
    whole = P // PAGE      # pages that all sequences have in common; a prefix that ends inside a page has a copy of it in each
    own_pages = [-(-(P + n) // PAGE) - whole for _, n in lengths]
    total = whole + sum(own_pages)
    order = torch.randperm(total, device="cuda", generator=g).int()
    tables = torch.full((len(lengths), whole + max(own_pages)), -1, dtype=torch.int32, device="cuda")
    at = whole
    for i, n in enumerate(own_pages):
        tables[i, :whole] = order[:whole]
        tables[i, whole:whole + n] = order[at:at + n]
        at += n
    k = torch.empty(total, nkv, PAGE, d, dtype=dtype, device="cuda").normal_(0, 1.3, generator=g)
    v = torch.empty(total, nkv, d, PAGE, dtype=dtype, device="cuda").normal_(0, 1, generator=g)
    rest = P - whole * PAGE
    if rest:
        first = tables[0, whole].long()
        for i in range(1, len(lengths)):
            k[tables[i, whole].long(), :, :rest] = k[first, :, :rest]
            v[tables[i, whole].long(), :, :, :rest] = v[first, :, :, :rest]
    T = sum(q for q, _ in lengths)
    q = torch.empty(T, case["heads"] * d, dtype=dtype, device="cuda").normal_(0, 1.3, generator=g)
    return {"q": q, "k": k, "v": v, "tables": tables}


def _verify_inputs(case, seed):
    """Logits of the target and of a drafter that is somewhat off, tokens drawn from the drafter (or guessed), random numbers."""
    g, V, drafts = _generator(seed), case["vocab"], _drafts(case)
    T = sum(drafts) + len(drafts)
    starts, at = [], 0
    for n in drafts:
        starts.append(at)
        at += n + 1
    logits = torch.empty(T, V, device="cuda").normal_(0, 2.5, generator=g)
    places = torch.tensor([s + j for s, n in zip(starts, drafts) for j in range(n)], device="cuda")      # rows that a draft is tested against
    tokens = torch.randint(0, V, (T,), device="cuda", generator=g, dtype=torch.int32)
    draft_logits = draft_rows = None
    rows = logits[places]
    if case["drafter"]:
        draft_logits = rows + torch.empty_like(rows).normal_(0, 0.5, generator=g)
        noise = torch.empty_like(rows).exponential_(generator=g).log_().neg_()
        tokens[places + 1] = (draft_logits / max(case["temperature"], 1e-3) + noise).argmax(-1).int()
        draft_rows = torch.full((T,), -1, dtype=torch.int32, device="cuda")
        draft_rows[places + 1] = torch.arange(len(places), device="cuda", dtype=torch.int32)
    else:       # three of four guesses are the target's first choice
        right = torch.rand(len(places), device="cuda", generator=g) < 0.75
        tokens[places + 1] = torch.where(right, rows.argmax(-1).int(), tokens[places + 1])
    del rows
    uniform = torch.rand(T, device="cuda", generator=g)
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    return {"logits": logits, "tokens": tokens, "starts": ints(starts), "lens": ints([n + 1 for n in drafts]), "uniform": uniform,
            "draft_logits": draft_logits, "draft_rows": draft_rows,
            "temperature": torch.full((len(drafts),), case["temperature"], device="cuda")}


def _q4_inputs(case, seed):
    """Codes 0 .. 15 (two a byte, the first in the low half) and scales of normal weights, rows of unit size."""
    g, N, K, group = _generator(seed), case["rows"], case["cols"], case["group"]
    codes = torch.empty(N, K // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(N, K // group, dtype=torch.bfloat16, device="cuda")
    for a in range(0, N, 8192):
        b = min(N, a + 8192)
        w = torch.empty(b - a, K // group, group, device="cuda").normal_(0, K ** -0.5, generator=g)
        s = (w.abs().amax(-1) / 7).bfloat16()
        c = ((w / s.float()[..., None]).round().clamp_(-8, 7) + 8).to(torch.uint8).view(b - a, K // 2, 2)
        codes[a:b], scales[a:b] = c[..., 0] | (c[..., 1] << 4), s
    x = torch.empty(case["tokens"], K, dtype=getattr(torch, case["dtype"]), device="cuda").normal_(0, 1, generator=g)
    return {"codes": codes, "scales": scales, "x": x}


def prepare(case, seed):
    state = {"shared": _shared_inputs, "verify": _verify_inputs, "q4": _q4_inputs}[case["op"]](case, seed)
    state["case"] = case
    if case["op"] == "shared":
        state["lengths"] = lengths = _lengths(case)
        state["out"] = torch.empty_like(state["q"])
        if not own:      # which row of the padded queries is which token
            most = max(q for q, _ in lengths)
            state["padded"] = torch.tensor([s * most + j for s, (q, _) in enumerate(lengths) for j in range(q)], device="cuda")
            state["last"] = torch.tensor([[n - q + j for j in range(most)] for q, n in lengths], device="cuda")      # own keys before a query
    if own:
        from sprout_lm_amd import ops
        if case["op"] == "shared":
            state["batch"] = ops.AttentionBatch.build([q for q, _ in lengths], [case["prefix"] + n for _, n in lengths], "cuda")
            kept = {}

            def workspace(n):
                if kept.get("t") is None or kept["t"].numel() < n:
                    kept["t"] = torch.empty(n, dtype=torch.float32, device="cuda")
                return kept["t"]
            state["workspace"] = workspace
        elif case["op"] == "verify":
            n = len(state["starts"])
            state["accepted"], state["next"] = (torch.empty(n, dtype=torch.int32, device="cuda") for _ in range(2))
            need = ops.verify_workspace_floats(len(state["logits"]), n, case["vocab"])
            state["workspace"] = torch.empty(need, dtype=torch.float32, device="cuda")
        else:
            state["w"] = ops.q4_pack(state.pop("codes"), state.pop("scales"), case["group"])
            state["out"] = torch.empty(case["tokens"], case["rows"], dtype=state["x"].dtype, device="cuda")
    return state


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    return {"shared": _run_shared, "verify": _run_verify, "q4": _run_q4}[state["case"]["op"]](state)


def _run_shared(state):
    c = state["case"]
    nq, nkv, d, P, scale = c["heads"], c["kv_heads"], c["dim"], c["prefix"], c["dim"] ** -0.5
    if own:
        from sprout_lm_amd import ops
        ops.attention_shared(state["q"], nq * d, state["k"], state["v"], state["tables"], state["batch"], P, state["out"], nq, nkv, d,
                             scale, workspace=state["workspace"])
        return state["out"]
    tables, lengths, G = state["tables"].long().clamp_min(0), state["lengths"], nq // nkv
    n, most, T = len(lengths), max(q for q, _ in lengths), len(state["q"])
    q = state["q"].float().view(T, nkv, G, d)
    # all queries by the prefix's keys: [kv heads, tokens * group, keys]
    pages = tables[0, :-(-P // PAGE)]
    k = state["k"][pages].float().permute(1, 0, 2, 3).reshape(nkv, -1, d)[:, :P]
    v = state["v"][pages].float().permute(1, 0, 3, 2).reshape(nkv, -1, d)[:, :P]
    far = torch.matmul(q.permute(1, 0, 2, 3).reshape(nkv, T * G, d), k.transpose(1, 2).contiguous()) * scale
    # every sequence's queries by its own keys, padded: [sequences, kv heads, queries * group, keys]
    first, longest = P // PAGE, max(m for _, m in lengths)
    skip = P - first * PAGE
    mine = tables[:, first:first + -(-(skip + longest) // PAGE)]
    own_k = state["k"][mine].float().permute(0, 2, 1, 3, 4).reshape(n, nkv, -1, d)[:, :, skip:skip + longest]
    own_v = state["v"][mine].float().permute(0, 2, 1, 4, 3).reshape(n, nkv, -1, d)[:, :, skip:skip + longest]
    padded = torch.zeros(n * most, nkv, G, d, device=q.device)
    padded[state["padded"]] = q
    padded = padded.view(n, most, nkv, G, d).permute(0, 2, 1, 3, 4).reshape(n, nkv, most * G, d)
    near = torch.matmul(padded, own_k.transpose(2, 3).contiguous()) * scale
    hidden = torch.arange(own_k.shape[2], device=q.device) > state["last"][:, :, None]
    near.masked_fill_(hidden[:, None, :, None].expand(n, 1, most, G, -1).reshape(n, 1, most * G, -1), -math.inf)
    near_top, far_top = near.amax(-1), far.amax(-1)
    near_w = torch.exp(near - near_top[..., None])
    near_o, near_l = torch.matmul(near_w, own_v), near_w.sum(-1)
    flat = lambda a: a.view(n, nkv, most, G, -1).permute(0, 2, 1, 3, 4).reshape(n * most, nkv, G, -1)[state["padded"]]
    near_o, near_l, near_top = flat(near_o), flat(near_l), flat(near_top)
    far_w = torch.exp(far - far_top[..., None])
    by_token = lambda a: a.view(nkv, T, G, -1).permute(1, 0, 2, 3)
    far_o, far_l, far_top = by_token(torch.matmul(far_w, v)), by_token(far_w.sum(-1)), by_token(far_top)
    top = torch.maximum(far_top, near_top)
    a, b = torch.exp(far_top - top), torch.exp(near_top - top)
    return ((far_o * a + near_o * b) / (far_l * a + near_l * b)).reshape(T, nq * d).to(state["q"].dtype)


def _run_verify(state):
    if own:
        from sprout_lm_amd import ops
        ops.verify_drafts(state["logits"], state["tokens"], state["starts"], state["lens"], state["uniform"], state["accepted"],
                          state["next"], state["workspace"], temperature=state["temperature"], draft_logits=state["draft_logits"],
                          draft_rows=state["draft_rows"])
        return state["accepted"], state["next"]
    # the answers are whole numbers next to borders: probabilities and sums in 64 bits
    logits, tokens, starts, lens, uniform = (state[k] for k in ("logits", "tokens", "starts", "lens", "uniform"))
    n, most = len(starts), state["case"]["drafts"]
    places = starts[:, None].long() + torch.arange(most, device=starts.device)      # rows that drafts are tested against
    there = torch.arange(most, device=starts.device) < lens[:, None] - 1
    places = torch.where(there, places, starts[:, None].long())
    drafted = tokens[(places + 1).clamp_max(len(tokens) - 1)].long()
    if state["case"]["temperature"] == 0.0:
        best = logits.argmax(-1)
        holds = (best[places] == drafted) & there
        accepted = holds.int().cumprod(-1).sum(-1)
        return accepted.int(), best[starts.long() + accepted].int()
    probabilities = lambda rows: torch.softmax(rows.double() / state["temperature"][0].double(), -1)
    p = probabilities(logits)
    p_d = p[places, drafted]
    if state["draft_logits"] is not None:
        q = probabilities(state["draft_logits"])
        q_row = state["draft_rows"][(places + 1).clamp_max(len(tokens) - 1)].long().clamp_min(0)
        q_d = q[q_row, drafted]
    else:
        q_d = torch.ones_like(p_d)
    holds = (uniform[places].double() * q_d < p_d) & there
    accepted = holds.int().cumprod(-1).sum(-1)
    last = starts.long() + accepted
    left, rejected = p[last], accepted < lens - 1
    which = accepted.clamp_max(most - 1)[:, None]
    if state["draft_logits"] is not None:
        off = q[q_row.gather(1, which)[:, 0]]
    else:
        off = torch.zeros_like(left).scatter_(1, drafted.gather(1, which), 1.0)
    left = torch.where(rejected[:, None], (left - off).clamp_min(0.0), left)
    running = left.cumsum(-1)
    limit = uniform[(starts + lens - 1).long()].double()[:, None] * running[:, -1:]
    return accepted.int(), (running <= limit).sum(-1).clamp_max(logits.shape[1] - 1).int()


def _run_q4(state):
    if own:
        from sprout_lm_amd import ops
        ops.gemm_q4(state["x"], state["w"], state["out"])
        return state["out"]
    codes, scales, x = state["codes"], state["scales"].float(), state["x"].float()
    N, K = codes.shape[0], 2 * codes.shape[1]
    w = torch.stack([codes & 15, codes >> 4], -1).view(N, scales.shape[1], -1).float()
    w = ((w - 8.0) * scales[..., None]).view(N, K)
    return torch.matmul(x, w.t()).to(state["x"].dtype)


# ---------------------------------------------------------------------------------------------- cost and truth
def work(case) -> dict:
    if case["op"] == "shared":
        lengths, element = _lengths(case), 2 if case["dtype"] == "bfloat16" else 4
        T, keys = sum(q for q, _ in lengths), case["prefix"] + sum(n for _, n in lengths)
        pairs = T * case["prefix"] + sum(q * n - q * (q - 1) // 2 for q, n in lengths)
        width = case["heads"] * case["dim"]
        return {"bytes": element * (2 * T * width + 2 * keys * case["kv_heads"] * case["dim"]), "flops": 4 * pairs * width}
    if case["op"] == "verify":
        drafts = _drafts(case)
        rows = sum(drafts) + len(drafts) + (sum(drafts) if case["drafter"] and case["temperature"] > 0 else 0)
        return {"bytes": 4 * rows * case["vocab"], "flops": (4 if case["temperature"] > 0 else 1) * rows * case["vocab"]}
    N, K, T = case["rows"], case["cols"], case["tokens"]
    element = 2 if case["dtype"] == "bfloat16" else 4
    return {"bytes": N * K // 2 + 2 * N * (K // case["group"]) + element * T * (K + N), "flops": 2 * T * N * K}


def exact(case, seed):
    """The definition in 64 bits, one sequence (of answers: one row) after the other."""
    if case["op"] == "shared":
        s = _shared_inputs(case, seed)
        nq, nkv, d, P = case["heads"], case["kv_heads"], case["dim"], case["prefix"]
        G, rows, at = nq // nkv, [], 0
        for i, (nq_i, n) in enumerate(_lengths(case)):
            ctx = P + n
            pages = s["tables"][i, :-(-ctx // PAGE)].long()
            k, v = s["k"][pages].double(), s["v"][pages].double()
            q = s["q"][at:at + nq_i].double().view(nq_i, nkv, G, d)
            at += nq_i
            heads = []
            for h in range(nkv):
                keys = k[:, h].reshape(-1, d)[:ctx]
                values = v[:, h].transpose(1, 2).reshape(-1, d)[:ctx]
                score = (q[:, h].reshape(-1, d) @ keys.t().contiguous()).view(nq_i, G, ctx) / math.sqrt(d)
                for j in range(nq_i):
                    score[j, :, ctx - nq_i + j + 1:] = -math.inf
                heads.append((torch.softmax(score, -1).view(-1, ctx) @ values).view(nq_i, G, d))
            rows.append(torch.stack(heads, 1).reshape(nq_i, nq * d))
        return torch.cat(rows)
    if case["op"] == "verify":
        s, accepted, following = _verify_inputs(case, seed), [], []
        for start, n in zip(s["starts"].tolist(), s["lens"].tolist()):
            tokens, u = s["tokens"][start:start + n].tolist(), s["uniform"][start:start + n].double().tolist()
            token = None
            for j in range(n):
                row, warmth = s["logits"][start + j].double(), case["temperature"]
                if warmth == 0.0:
                    best = int(row.argmax())
                    if j < n - 1 and tokens[j + 1] == best:
                        continue
                    token = best
                    break
                p = torch.exp(row / float(s["temperature"][0]) - torch.logsumexp(row / float(s["temperature"][0]), 0))
                if j < n - 1:
                    if s["draft_logits"] is not None:
                        other = s["draft_logits"][int(s["draft_rows"][start + j + 1])].double() / float(s["temperature"][0])
                        q = torch.exp(other - torch.logsumexp(other, 0))
                    else:
                        q = torch.zeros_like(p)
                        q[tokens[j + 1]] = 1.0
                    if u[j] * float(q[tokens[j + 1]]) < float(p[tokens[j + 1]]):
                        continue
                    p = (p - q).clamp_min(0.0)
                running = torch.cumsum(p, 0)
                token = min(int(torch.searchsorted(running, running[-1] * u[n - 1], right=True)), len(p) - 1)
                break
            accepted.append(j)
            following.append(token)
        as_ints = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
        return as_ints(accepted), as_ints(following)
    s, N, K = _q4_inputs(case, seed), case["rows"], case["cols"]
    x, parts = s["x"].double(), []
    for a in range(0, N, 4096):
        codes = s["codes"][a:a + 4096]
        w = torch.empty(len(codes), K, dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = (codes & 15).double() - 8, (codes >> 4).double() - 8
        w *= s["scales"][a:a + 4096].double().repeat_interleave(case["group"], 1)
        parts.append(x @ w.t().contiguous())
    return torch.cat(parts, 1)

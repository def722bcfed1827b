"""Scoring of given tokens: from request lengths to the tables of a step, and from logits or hidden states to log-probabilities.

Three operators of `xllm_b200.ops`:

  token   `score.token_logprobs`: log-probability of a given token, entropy and the most likely alternatives of every row of
          logits, under an optional temperature per row
  head    `score.head_logprobs`: log-probability and entropy straight from hidden states and the output projection
  tables  `tables.step_tables`: row ranges, lengths, positions, cache slots and newly taken cache blocks of a step

`run` computes them in plain torch, or through the framework where `own` is set.
"""
import math

import numpy as np
import torch

own = False

MOST_ELEMENTS = 4000 * 151936          # logits of the largest listed case
MOST_SORTED = 1000 * 151936            # ... of the largest one that lists alternatives


# ----------------------------------------------------------------------------- the cases
def _token(name, rows, vocab, dtype="bfloat16", n_top=0, temperature=False, kept=1.0, pad=0):
    return {"name": name, "op": "token", "rows": rows, "vocab": vocab, "dtype": dtype, "n_top": n_top, "temperature": temperature,
            "kept": kept, "pad": pad}


def _head(name, rows, width, vocab, temperature=False):
    return {"name": name, "op": "head", "rows": rows, "width": width, "vocab": vocab, "temperature": temperature}


def _tables(name, requests, context, new, page, scarce=False):
    return {"name": name, "op": "tables", "requests": requests, "context": context, "new": new, "page": page, "scarce": scarce}


def listed():
    return [
        _token("token_one_row", 1, 151936, n_top=5),                              # one user asks for alternatives: latency
        _token("token_decode", 64, 151936, n_top=20, temperature=True),           # a busy server, most alternatives the API gives
        _token("token_masked_f32", 500, 32003, "float32", n_top=1, kept=0.3, pad=5),   # grammar masks, fp32 rows of a wider buffer
        _token("token_alternatives", 1000, 151936, n_top=5),                      # a prompt scored with alternatives
        _token("token_prompt", 4000, 151936),                                     # a long prompt scored, no alternatives
        _head("head_one_row", 1, 4096, 151936),                                   # one row against the whole projection
        _head("head_choices", 45, 2048, 151936, temperature=True),                # short answers ranked by likelihood
        _head("head_prompt", 1000, 4096, 32768),                                  # a prompt, small vocabulary
        _head("head_batch", 4096, 4096, 151936),                                  # a batch of prompts scored
        _tables("tables_decode", 64, 4000, 1, 16),                                # a decode step: one token a request
        _tables("tables_prompts", 13, 700, 1200, 64),                             # prompt portions behind cached prefixes
        _tables("tables_offline", 3000, 900, 150, 16, scarce=True),               # an offline queue, more than the blocks hold
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    op = rng.choice(["token", "token", "head", "head", "tables"])
    if op == "token":
        vocab = rng.choice([32000, 32768, 50257, 129280, 151936, log(300, 151936)])
        dtype, n_top = rng.choice(["bfloat16", "bfloat16", "float32"]), rng.choice([0, 0, 1, 5, 20, rng.randint(2, 64)])
        most = (MOST_SORTED if n_top else MOST_ELEMENTS) // vocab // (2 if dtype == "float32" else 1)
        case = _token("", log(1, min(4000, most)), vocab, dtype, n_top, rng.random() < 0.5, rng.choice([1.0, 1.0, 0.5]),
                      rng.choice([0, 0, rng.randint(1, 40)]))
    elif op == "head":
        case = _head("", log(1, 4096), rng.choice([512, 1024, 2048, 2880, 4096, 8 * log(16, 512)]),
                     rng.choice([32000, 32768, 50257, 129280, 151936, log(300, 151936)]), rng.random() < 0.5)
    else:
        requests = log(1, 3000)
        new = max(1, min(rng.choice([1, 1, log(2, 2000)]), 450000 // requests))
        case = _tables("", requests, log(1, 8000) if requests < 500 else log(1, 1500), new,
                       rng.choice([1, 16, 32, 64, 128]) if new < 200 else 64, rng.random() < 0.25)
    del case["name"]
    return case


# ----------------------------------------------------------------------------- inputs
def _generator(seed, device):
    g = torch.Generator(device=device)
    g.manual_seed(seed * 7919 + 17)
    return g


def _temperature(case, g, device):
    """Sampling temperatures of a batch: most requests set one, some leave it at 0 (greedy, read as 1)."""
    if not case["temperature"]:
        return None
    t = torch.empty(case["rows"], device=device).uniform_(0.4, 1.4, generator=g)
    t[::7] = 0.0
    return t


def _prepare_token(case, seed, device):
    g = _generator(seed, device)
    B, V, dt = case["rows"], case["vocab"], getattr(torch, case["dtype"])
    logits = torch.empty((B, V + case["pad"]), dtype=dt, device=device).normal_(0.0, 2.0, generator=g)[:, :V]
    ids = torch.randint(0, V, (B,), generator=g, device=device)
    peak = torch.empty((B, 1), device=device).uniform_(0.0, 14.0, generator=g)        # a model is sure of some places only
    logits.scatter_(1, ids[:, None], peak.to(dt))
    if case["kept"] < 1.0:
        barred = torch.rand((B, V), generator=g, device=device) >= case["kept"]
        barred.scatter_(1, ids[:, None], False)
        logits.masked_fill_(barred, float("-inf"))
    ids[5::11] = -1                                                                  # places nobody asks about
    return {"op": "token", "logits": logits, "ids": ids, "n_top": case["n_top"], "temperature": _temperature(case, g, device)}


def _prepare_head(case, seed, device):
    g = _generator(seed, device)
    T, K, V = case["rows"], case["width"], case["vocab"]
    weight = torch.empty((V, K), dtype=torch.bfloat16, device=device).normal_(0.0, 1.4 / math.sqrt(K), generator=g)
    ids = torch.randint(0, V, (T,), generator=g, device=device)
    hidden = torch.empty((T, K), device=device).normal_(0.0, 1.0, generator=g)
    sure = torch.empty((T, 1), device=device).uniform_(0.0, 4.0, generator=g)         # final states point at the next token
    hidden = (hidden + sure * weight[ids].float()).to(torch.bfloat16)
    ids[5::11] = -1
    return {"op": "head", "hidden": hidden, "weight": weight, "ids": ids, "temperature": _temperature(case, g, device)}


def _lengths(case, seed):
    """(context lengths, new tokens) of the requests: ragged, some contexts empty, some a whole number of blocks."""
    rng = np.random.default_rng(seed * 31 + 5)
    B = case["requests"]
    ctx = np.maximum(0, np.round(case["context"] * (1.0 - 0.75 * rng.random(B)))).astype(np.int64)
    if case["new"] > 1:
        ctx[1::4] = 0
    ctx[2::8] -= ctx[2::8] % case["page"]
    # the same lengths for every seed, handed to the requests in another order: a step has so many token rows
    share = 1.0 - 0.8 * ((np.arange(B) * 0.6180339887) % 1.0)
    new = rng.permutation(np.maximum(1, np.round(case["new"] * share)).astype(np.int64)) if case["new"] > 1 else np.ones(B, np.int64)
    return ctx, new


def _pool(case, seed):
    """Host side of a step: the block table before it, the free blocks in the order they are handed out, the table's width."""
    ctx, new = _lengths(case, seed)
    rng = np.random.default_rng(seed * 37 + 11)
    page = case["page"]
    have, need = -(-ctx // page), -(-(ctx + new) // page)
    width = int(-(-(case["context"] + case["new"]) // page)) + 1
    total, added = int(have.sum()), int((need - have).sum())
    order = rng.permutation(total + added + 4096).astype(np.int32)        # the cache is larger than these requests
    table = np.full((case["requests"], width), -1, np.int32)
    table[np.arange(width)[None, :] < have[:, None]] = order[:total]
    n_free = int(added * 0.9) if case["scarce"] else added + 8
    return ctx, new, table, order[total:total + n_free]


def _prepare_tables(case, seed, device):
    ctx, new, table, free = _pool(case, seed)
    to = lambda a, dt: torch.from_numpy(np.ascontiguousarray(a)).to(device=device, dtype=dt)
    return {"op": "tables", "block_table": to(table, torch.int32), "ctx_lens": to(ctx, torch.int32), "q_lens": to(new, torch.int32),
            "free_blocks": to(free, torch.int32), "page": case["page"], "n_rows": int(new.sum()) + 3}


def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    return {"token": _prepare_token, "head": _prepare_head, "tables": _prepare_tables}[case["op"]](case, seed, device)


# ----------------------------------------------------------------------------- the plain forms
def _plain_token(x, ids, n_top, temperature):
    x = x.float()
    u = x if temperature is None else x / torch.where(temperature > 0, temperature, 1.0)[:, None]
    m = u.amax(1, keepdim=True)
    m = torch.where(m == float("-inf"), 0.0, m)
    d = u - m
    e = torch.exp(d)
    z = e.sum(1)
    log_z = torch.log(z)
    entropy = log_z - torch.where(e > 0, e * d, 0.0).sum(1) / z
    logprob = torch.where(ids >= 0, d.gather(1, ids.clamp(min=0)[:, None])[:, 0] - log_z, 0.0)
    if n_top == 0:
        return logprob, entropy
    top = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :n_top]
    return logprob, entropy, top.to(torch.int32), d.gather(1, top) - log_z[:, None]


def _plain_tables(s):
    table, page, rows = s["block_table"], s["page"], s["n_rows"]
    ctx, new, free = s["ctx_lens"].long(), s["q_lens"].long(), s["free_blocks"]
    B, width = table.shape
    end = torch.cumsum(new, 0)
    have, need = (ctx + page - 1) // page, (ctx + new + page - 1) // page
    fits = (need <= width) & (end <= rows)
    added = torch.where(fits, need - have, 0)
    upto = torch.cumsum(added, 0)
    ok = fits & ((added == 0) | (upto <= free.shape[0]))
    taken = torch.where(ok, added, 0).sum()

    block = torch.arange(free.shape[0], device=table.device)
    owner = torch.searchsorted(upto, block, right=True).clamp(max=B - 1)
    column = have[owner] + block - (upto - added)[owner]
    cells = torch.cat([table.flatten(), table.new_zeros(1)])            # the last cell takes what is not handed out
    cells[torch.where(block < taken, owner * width + column, B * width)] = free
    table.copy_(cells[:-1].view(B, width))

    row = torch.arange(rows, device=table.device)
    seq = torch.searchsorted(end, row, right=True).clamp(max=B - 1)
    live = (row < end[-1]) & ok[seq]
    positions = torch.where(live, ctx[seq] + row - (end - new)[seq], 0)
    entry = table[seq, (positions // page).clamp(max=width - 1)].long()
    slots = torch.where(live, entry * page + positions % page, -1)
    cu_q = torch.cat([end.new_zeros(1), end.clamp(max=rows)])
    return (cu_q.int(), torch.where(ok, ctx + new, 0).int(), positions, slots.int(), (cu_q[1:] - 1).clamp(min=0), taken.int(), table)


def run(s):
    if s["op"] == "token":
        if own:
            from xllm_b200.ops import score
            out = score.token_logprobs(s["logits"], s["ids"], s["n_top"], temperature=s["temperature"])
            return out if s["n_top"] else out[:2]
        return _plain_token(s["logits"], s["ids"], s["n_top"], s["temperature"])
    if s["op"] == "head":
        if own:
            from xllm_b200.ops import score
            return score.head_logprobs(s["hidden"], s["weight"], s["ids"], temperature=s["temperature"])
        return _plain_token(s["hidden"].float() @ s["weight"].float().T, s["ids"], 0, s["temperature"])
    if own:
        from xllm_b200.ops import tables
        t = tables.step_tables(s["block_table"], s["ctx_lens"], s["q_lens"], s["page"], s["n_rows"], s["free_blocks"])
        return t.cu_q, t.kv_lens, t.positions, t.slots, t.last_rows, t.taken, s["block_table"]
    return _plain_tables(s)


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "token":
        B, V = case["rows"], case["vocab"]
        return {"bytes": B * V * (2 if case["dtype"] == "bfloat16" else 4) + B * (16 + 8 * case["n_top"]), "flops": 5 * B * V}
    if case["op"] == "head":
        T, K, V = case["rows"], case["width"], case["vocab"]
        return {"bytes": 2 * K * (T + V) + 16 * T, "flops": 2 * T * K * V + 5 * T * V}
    ctx, new = _lengths(case, 1)
    rows, added = int(new.sum()), int((-(-(ctx + new) // case["page"]) - -(-ctx // case["page"])).sum())
    # lengths in; ranges, lengths and last rows out; a position and a slot a row; new blocks read and written; the first entry read
    return {"bytes": case["requests"] * (8 + 4 + 4 + 8 + 4) + 12 * rows + 8 * added, "flops": 4 * rows}


# ----------------------------------------------------------------------------- in 64 bits, from the definitions
def _exact_rows(x, ids, temperature, n_top):
    """One chunk of rows of fp64 scores."""
    scaled = x if temperature is None else x / torch.where(temperature > 0, temperature.double(), 1.0)[:, None]
    p = torch.softmax(scaled, dim=1)
    lse = torch.logsumexp(scaled, dim=1)
    entropy = -torch.special.xlogy(p, p).sum(1)
    asked = ids >= 0
    logprob = torch.zeros_like(lse)
    logprob[asked] = scaled[asked].gather(1, ids[asked][:, None])[:, 0] - lse[asked]
    if n_top == 0:
        return logprob, entropy
    # the order of (score, lowest index first) as whole numbers: the bits of an fp32 score in ascending order, then the index
    bits = (x.float() + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 20) - torch.arange(x.shape[1], device=x.device)
    top = order.topk(n_top, dim=1).indices
    return logprob, entropy, top, scaled.gather(1, top) - lse[:, None]


def _exact_scores(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    if case["op"] == "token":
        s = _prepare_token(case, seed, device)
        rows, scores = s["logits"], lambda c: c.double()
    else:
        s = _prepare_head(case, seed, device)
        wide = s["weight"].double()
        rows, scores = s["hidden"], lambda c: c.double() @ wide.T
    parts = []
    for at in range(0, rows.shape[0], 256):
        cut = slice(at, at + 256)
        t = None if s["temperature"] is None else s["temperature"][cut]
        parts.append(_exact_rows(scores(rows[cut]), s["ids"][cut], t, case.get("n_top", 0)))
    return tuple(torch.cat(p) for p in zip(*parts))


def _exact_tables(case, seed):
    ctx, new, table, free = _pool(case, seed)
    page, width, rows = case["page"], table.shape[1], int(new.sum()) + 3
    positions, slots = np.zeros(rows, np.int64), np.full(rows, -1, np.int64)
    cu, lens, last, at, spent, taken = [0], [], [], 0, 0, 0
    for b, (c, q) in enumerate(zip(ctx.tolist(), new.tolist())):
        have, need = (c + page - 1) // page, (c + q + page - 1) // page
        start, at = at, at + q
        fits = need <= width and at <= rows
        add = need - have if fits else 0
        spent += add
        ok = fits and (add == 0 or spent <= len(free))
        if ok:
            table[b, have:need] = free[spent - add:spent]
            taken += add
            pos = np.arange(c, c + q)
            positions[start:at], slots[start:at] = pos, table[b, pos // page].astype(np.int64) * page + pos % page
        cu.append(min(at, rows))
        lens.append(c + q if ok else 0)
        last.append(max(cu[-1] - 1, 0))
    return tuple(torch.from_numpy(np.asarray(v)) for v in (cu, lens, positions, slots, last, taken, table))


def exact(case, seed):
    return _exact_tables(case, seed) if case["op"] == "tables" else _exact_scores(case, seed)

"""Log-probabilities of given tokens: what a model thinks of text it did not write (perplexity, choice by likelihood, re-scoring).

Prompts are packed into ragged passes on a scratch cache, like embedding requests never in the serving pool.  The tables of a
pass are built on the device from the prompts' lengths (ops/tables.py); its final hidden states are scored without ever holding
the logits (ops.score.head_logprobs).  Alternatives, where asked for, come from logits in portions of rows, rounded like those that
tokens are sampled from; the scores are the same with and without them.
"""
from __future__ import annotations

from typing import List, NamedTuple, Optional

import torch

from ..engine.model_runner import ModelRunner
from ..models.layers import AttentionMetadata
from ..ops import score, tables

LOGIT_ROWS = 256            # rows whose logits are held at a time
HEAD_ROWS = 8192            # rows whose tallies are: 78 MB of them for 151936 tokens


class TokenScores(NamedTuple):
    """Of one prompt, an entry per token; those of the first token are None: nothing comes before it."""
    logprobs: List[Optional[float]]
    entropies: List[Optional[float]]                    # of the distribution that the token was picked from, in nats
    top_logprobs: Optional[List[Optional[List[tuple]]]]  # [(token id, logprob), ...] most likely first; of logits as they are sampled from


def _scratch_cache(engine, n_blocks):
    out = []
    for g in ModelRunner.kv_layout(engine.model, engine.args):
        kv = None if g is None else torch.zeros(g[0], n_blocks, g[1], engine.cfg.block_size, g[2], dtype=engine.dtype, device=engine.device)
        out.append((None, None) if kv is None else (kv[0], kv[g[0] - 1]))
    return out


def _passes(lengths, limit, whole):
    """Groups of prompts that share a cache, each a list of passes [(prompt, first token, tokens), ...]: as many short prompts as
    fit `limit` tokens in one pass, a longer one by itself in several, or in one where `whole` and then with no other."""
    groups, open_, n = [], [], 0
    for i, L in enumerate(lengths):
        if L == 0:
            continue
        if whole or L > limit:
            step = L if whole else limit
            groups.append([[(i, at, min(step, L - at))] for at in range(0, L, step)])
            continue
        if n + L > limit or len(open_) == tables.MAX_REQUESTS:
            groups.append([open_])
            open_, n = [], 0
        open_.append((i, 0, L))
        n += L
    return groups + ([[open_]] if open_ else [])


def _forward(engine, prompts, work, table, free, cache):
    """Final hidden states [tokens, width] of one pass."""
    model, dev = engine.model, engine.device
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    tokens = [t for i, at, n in work for t in prompts[i][at:at + n]]
    step = tables.step_tables(table, i32([at for _, at, _ in work]), i32([n for _, _, n in work]), engine.cfg.block_size, len(tokens), free)
    meta = AttentionMetadata(n_decode=0, n_prefill=len(work), slots=step.slots, block_table=table, kv_lens=step.kv_lens, cu_q=step.cu_q,
                             max_q_len=max(n for _, _, n in work), max_kv_len=max(at + n for _, at, n in work))
    if getattr(model, "needs_state", False):            # a scratch state slot, reset for this pass
        meta.state_slots = torch.tensor([model.state.scratch_slot], device=dev,
                                        dtype=torch.int32 if getattr(model, "state_on_device", False) else torch.long)
        meta.state_fresh, meta.seq_bounds = [True], [(0, len(tokens))]
    return model.forward(torch.tensor(tokens, dtype=torch.int64, device=dev), step.positions, meta, cache)


def _score_rows(model, hidden, targets, n_top, temperature):
    head = model.lm_head
    weight = head.weight[:head.vocab]
    t = None if temperature is None else torch.full((hidden.shape[0],), temperature, dtype=torch.float32, device=hidden.device)
    fused = score.head_supported(hidden, weight)

    def portions(rows):
        return [(hidden[at:at + rows], targets[at:at + rows], None if t is None else t[at:at + rows]) for at in range(0, hidden.shape[0], rows)]
    from_head = [score.head_logprobs(h, weight, ids, temperature=T) for h, ids, T in portions(HEAD_ROWS)] if fused else []
    from_logits = [score.token_logprobs(model.logits(h), ids, n_top, temperature=T) for h, ids, T in portions(LOGIT_ROWS)] \
        if n_top or not fused else []
    scores = [torch.cat(p) for p in list(zip(*(from_head or from_logits)))[:2]]
    return scores + ([torch.cat(p) for p in list(zip(*from_logits))[2:]] if n_top else [None, None]), fused


def score_token_lists(engine, prompts: List[List[int]], n_top: int = 0, temperature: Optional[float] = None) -> List[TokenScores]:
    """Scores of every token of every prompt (token ids), with `n_top` alternatives each, under softmax(logits / temperature).
    RuntimeError where a wait of a kernel expired: its scores are not there."""
    out, passes = score_in_passes(engine, prompts, n_top, temperature)
    for _ in passes:
        pass
    return out


def score_in_passes(engine, prompts, n_top=0, temperature=None):
    """(scores, passes) of `score_token_lists`: what is asked for is checked here; the scores are filled in while `passes` is gone
    through, a pass of the model each, between which the engine may step."""
    model, vocab = engine.model, engine.model.lm_head.vocab
    if engine.asleep:
        raise RuntimeError("the engine is asleep")
    if engine.ps.world_size > 1:
        raise ValueError("scoring runs on one rank: the passes are not scheduled over several")
    if getattr(model, "needs_index_cache", False):
        raise ValueError("scoring needs a scratch cache for everything a model keeps per token: this one has an index cache of its own")
    if not 0 <= n_top <= min(score.MAX_TOP, vocab):
        raise ValueError(f"0 to {min(score.MAX_TOP, vocab)} alternatives, asked for {n_top}")
    if temperature is not None and not 1e-6 <= temperature <= 1e6:      # results stay finite, as JSON needs them
        raise ValueError(f"a temperature of 1e-6 to 1e6, not {temperature}")
    for p in prompts:
        if len(p) > engine.max_model_len:
            raise ValueError(f"a prompt of {len(p)} tokens, the model takes {engine.max_model_len}")
        if any(not 0 <= t < vocab for t in p):
            raise ValueError(f"token ids are 0 to {vocab - 1}")
    out = [TokenScores([None] * min(len(p), 1), [None] * min(len(p), 1), [None] * min(len(p), 1) if n_top else None) for p in prompts]
    return out, _run_passes(engine, prompts, n_top, temperature, out)


@torch.no_grad()
def _run_passes(engine, prompts, n_top, temperature, out):
    model, page, dev = engine.model, engine.cfg.block_size, engine.device
    whole = bool(getattr(model, "needs_state", False))
    for group in _passes([len(p) for p in prompts], engine.cfg.max_tokens_per_batch, whole):
        longest = max(at + n for work in group for _, at, n in work)
        blocks = sum(-(-len(prompts[i]) // page) for i, _, _ in group[-1])
        cache = _scratch_cache(engine, blocks)
        free = torch.arange(blocks, dtype=torch.int32, device=dev)
        table = torch.zeros(len(group[0]), -(-longest // page), dtype=torch.int32, device=dev)
        for work in group:
            if engine.asleep:
                raise RuntimeError("the engine is asleep")
            taken = -(-work[0][1] // page)              # blocks of the passes before; 0 where the pass holds several prompts
            hidden = _forward(engine, prompts, work, table, free[taken:], cache)
            given = [t for i, at, n in work for t in (prompts[i] + [-1])[at + 1:at + n + 1]]
            results, fused = _score_rows(model, hidden, torch.tensor(given, dtype=torch.int64, device=dev), n_top, temperature)
            lps, ents, top, top_lps = [None if r is None else r.tolist() for r in results]
            if fused and score.expired():              # behind the copies that waited for it
                raise RuntimeError("a bounded wait inside head_logprobs expired: no scores")
            row = 0
            for i, at, n in work:
                m = min(n, len(prompts[i]) - 1 - at)    # the row of a prompt's last token has nothing to score
                out[i].logprobs.extend(lps[row:row + m])
                out[i].entropies.extend(ents[row:row + m])
                if n_top:
                    out[i].top_logprobs.extend([[(t, v) for t, v in zip(a, b) if t >= 0]
                                                for a, b in zip(top[row:row + m], top_lps[row:row + m])])
                row += n
            yield

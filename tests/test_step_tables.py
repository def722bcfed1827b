"""Tables of a step from request lengths (`ops.tables`) against a plain loop over requests and tokens."""
import random

import pytest
import torch

from xllm_b200.ops import tables

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def plain(table, ctx, new, page, n_rows, free):
    """The contract, one request and one token at a time; `table` (lists) is updated."""
    cu, lens, pos, slots, last, spent, taken = [0], [], [0] * n_rows, [-1] * n_rows, [], 0, 0
    at = 0
    for b, (c, q) in enumerate(zip(ctx, new)):
        c, q = max(c, 0), max(q, 0)
        have, need = -(-c // page), -(-(c + q) // page)
        start, at = at, at + q
        ok = need <= len(table[b]) and at <= n_rows and c + q < 1 << 31
        if ok:
            spent += need - have
            ok = need == have or spent <= len(free)
        if ok:
            for j in range(have, need):
                table[b][j] = free[spent - (need - have) + j - have]
            taken += need - have
            for i in range(q):
                pos[start + i] = c + i
                block = table[b][(c + i) // page]
                slot = block * page + (c + i) % page
                slots[start + i] = slot if block >= 0 and slot < 1 << 31 else -1
        cu.append(min(at, n_rows))
        lens.append(c + q if ok else 0)
        last.append(max(cu[-1] - 1, 0))
    return cu, lens, pos, slots, last, taken


def check(ctx, new, page, device, width=None, n_rows=None, free=None, pad=0, seed=0):
    rng = random.Random(seed)
    B = len(ctx)
    need = [-(-(max(c, 0) + max(q, 0)) // page) for c, q in zip(ctx, new)]
    width = width or max(need + [1]) + 1
    n_rows = sum(max(q, 0) for q in new) + pad if n_rows is None else n_rows
    names = list(range(5, 5 + sum(need) + 40))
    rng.shuffle(names)
    table = [[-7] * width for _ in range(B)]
    for b in range(B):
        for j in range(min(width, -(-max(ctx[b], 0) // page))):
            table[b][j] = names.pop()
    free = names[:sum(need) + 3] if free is None else names[:free]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
    whole = torch.full((B, width + 3), -9, dtype=torch.int32, device=device)
    whole[:, :width] = i32(table)
    got = tables.step_tables(whole[:, :width], i32(ctx), i32(new), page, n_rows, i32(free) if free else None)
    want = plain(table, ctx, new, page, n_rows, free)
    for name, a, w in zip(got._fields, got, want):
        assert a.cpu().tolist() == w, name
    assert [t.dtype for t in got] == [torch.int32, torch.int32, torch.int64, torch.int32, torch.int64, torch.int32]
    assert whole[:, :width].cpu().tolist() == table
    assert bool((whole[:, width:] == -9).all())
    return got


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("page", [1, 16, 64, 7])
@pytest.mark.parametrize("ctx,new", [([0], [1]), ([0], [40]), ([15], [1]), ([16], [1]), ([17, 0, 64], [1, 1, 1]), ([0, 0, 0], [0, 0, 0]),
                                     ([5, 0, 32, 100], [0, 33, 64, 1]), ([0, 3, 0], [0, 1, 0]), ([100, 3], [500, 1000]), ([-4, 8], [3, -2])])
def test_small(device, page, ctx, new):
    check(ctx, new, page, device)
    check(ctx, new, page, device, pad=29)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("B", [2, 31, 33, 500, 513, 1025, 3000])
@pytest.mark.parametrize("decode", [True, False])
def test_ragged(device, B, decode):
    rng = random.Random(B)
    ctx = [rng.choice([0, rng.randint(0, 300), 64 * rng.randint(0, 4)]) for _ in range(B)]
    new = [1 if decode else rng.choice([0, 1, rng.randint(1, 60)]) for _ in range(B)]
    for page in (16, 64):
        check(ctx, new, page, device, pad=rng.choice([0, 5]), seed=B)


@pytest.mark.parametrize("device", DEVICES)
def test_short_of_blocks(device):
    ctx, new = [10, 0, 30, 16, 0, 5], [10, 40, 2, 1, 33, 1]
    for free in range(0, 9):
        got = check(ctx, new, 16, device, free=free)
        assert int(got.taken) <= free
    assert check(ctx, new, 16, device, free=1).kv_lens.tolist() == [20, 0, 32, 0, 0, 6]


@pytest.mark.parametrize("device", DEVICES)
def test_short_of_rows_and_width(device):
    ctx, new = [10, 0, 30, 16, 0, 5], [10, 40, 2, 1, 33, 1]
    for n_rows in (0, 1, 9, 10, 11, 49, 50, 52, 53, 85, 86, 87):
        check(ctx, new, 16, device, n_rows=n_rows)
    for width in (1, 2, 3):
        check(ctx, new, 16, device, width=width)


@pytest.mark.parametrize("device", DEVICES)
def test_far_positions(device):
    """Lengths whose sum passes 31 bits are refused, not wrapped; slots behind 31 bits are not written."""
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
    table = i32([[3, 4, 5], [6, 7, 8]])
    got = tables.step_tables(table, i32([2 ** 31 - 1, 2 ** 30 + 5]), i32([5, 3]), 2 ** 30, 10, None)
    assert got.kv_lens.tolist() == [0, 2 ** 30 + 8] and got.positions.tolist() == [0] * 5 + [2 ** 30 + 5 + i for i in range(3)] + [0] * 2
    assert got.slots.tolist() == [-1] * 10
    assert table.tolist() == [[3, 4, 5], [6, 7, 8]]
    many = i32([2 ** 31 - 1] * 4)
    got = tables.step_tables(i32([[1]] * 4), i32([0] * 4), many, 2 ** 31 - 1, 7, None)
    assert got.cu_q.tolist() == [0, 7, 7, 7, 7] and got.kv_lens.tolist() == [0] * 4 and int(got.taken) == 0


@pytest.mark.gpu
def test_largest():
    B = tables.MAX_REQUESTS
    rng = random.Random(1)
    ctx, new = [rng.randint(0, 40) for _ in range(B)], [rng.randint(0, 3) for _ in range(B)]
    check(ctx, new, 16, "cuda", pad=1)
    check([0], [300000], 1, "cuda")


@pytest.mark.gpu
def test_most_requests_first():
    """Numbers of requests around the shared memory that a launch gets without asking, in a process that has had no larger call."""
    import os
    import subprocess
    import sys
    code = f"""
import sys
sys.path.insert(0, {os.path.dirname(os.path.abspath(__file__))!r})
from test_step_tables import check
for B in (4053, 4074, 4075, 4090, 4096, 4097):
    check([b % 40 for b in range(B)], [b % 3 for b in range(B)], 16, "cuda", pad=1)
print("served")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "served" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("width", [1 << 31, (1 << 32) + 5])
def test_too_wide(width):
    """More entries than a kernel counts in 32 bits; nothing of them is read."""
    e = lambda *shape: torch.empty(*shape, dtype=torch.int32, device="meta")
    with pytest.raises(ValueError, match="width"):
        tables.step_tables(e(1, width), e(1), e(1), 16, 4, e(3))


def test_refusals():
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    ok = dict(block_table=i32(2, 3), ctx_lens=i32(2), q_lens=i32(2), page=16, n_rows=4, free_blocks=i32(5))
    tables.step_tables(**ok)
    for change, error in ((dict(block_table=i32(2, 3).long()), TypeError), (dict(block_table=i32(3, 2).T), TypeError),
                          (dict(ctx_lens=i32(3)), TypeError), (dict(q_lens=i32(2).long()), TypeError), (dict(free_blocks=i32(5).long()), TypeError),
                          (dict(free_blocks=i32(5, 1)), TypeError), (dict(free_blocks=i32(1).expand(1 << 32)), TypeError),
                          (dict(page=0), ValueError), (dict(page=(1 << 32) + 16), ValueError), (dict(n_rows=-1), ValueError),
                          (dict(block_table=i32(1, 3).expand(2, -1)), ValueError), (dict(block_table=i32(2, 0)), ValueError), (dict(block_table=i32(0, 3), ctx_lens=i32(0), q_lens=i32(0)), ValueError),
                          (dict(block_table=i32(8193, 1), ctx_lens=i32(8193), q_lens=i32(8193)), ValueError)):
        with pytest.raises(error):
            tables.step_tables(**{**ok, **change})


@pytest.mark.gpu
def test_captured_decode_steps():
    """A captured step replayed with the lengths that the step before left: every request gets its blocks as it grows."""
    B, page, width, steps = 6, 4, 8, 9
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    table, ctx, one = torch.full((B, width), -1, dtype=torch.int32, device="cuda"), i32([0] * B), i32([1] * B)
    free, out = i32(list(range(100, 160))), []
    tables.step_tables(table.clone(), ctx, one, page, B + 2, free)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        t = tables.step_tables(table, ctx, one, page, B + 2, free)
        ctx.copy_(t.kv_lens)
    for s in range(steps):
        g.replay()
        torch.cuda.synchronize()
        assert t.positions.tolist() == [s] * B + [0, 0] and t.kv_lens.tolist() == [s + 1] * B
        assert int(t.taken) == (B if s % page == 0 else 0)
        assert t.slots.tolist() == [table[b, s // page].item() * page + s % page for b in range(B)] + [-1, -1]
        if int(t.taken):
            free.copy_(torch.roll(free, -int(t.taken)))
    used = table[:, :3].flatten().tolist()
    assert sorted(used) == list(range(100, 100 + 3 * B))

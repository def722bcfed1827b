"""Scoring of given tokens (`ops.score`) against plain formulas in 64 bits.

Bounds.  With u = (x - max x) / T and z = sum exp u, an fp32 result carries: the roundings of u (difference, factor, product)
and of the last sum and product, 6 x 2^-24 of |u| + log z; of an exponential 2^-22 and what its argument is off by; of a sum
at most one rounding an addition, and no accumulator takes more than a 128th of a row.  So the log-probability is off by at
most 2^-24 (V / 128 + 64) (1 + |u| + log V), and the entropy, whose terms are probabilities times |u|, by twice that.
"""
import math

import pytest
import torch

from xllm_b200.ops import score

STEP = 2.0 ** -24


def exact(x, ids, n_top=0, temperature=None):
    """(logprob, entropy, alternatives, their log-probabilities, |u| of the given tokens) in 64 bits, a row at a time."""
    lps, ents, tops, top_lps, far = [], [], [], [], []
    V = x.shape[1]
    for r in range(x.shape[0]):
        row, i = x[r].double().cpu(), int(ids[r])
        T = 1.0 if temperature is None or not float(temperature[r]) > 0 else float(temperature[r])
        bad = bool(torch.isnan(row).any()) or bool((row == math.inf).any())
        live = row[~torch.isnan(row)]
        none = not bad and bool((row == -math.inf).all())
        m = 0.0 if none else (float(live.max()) if len(live) else 0.0)
        u = (row - m) / T
        z = torch.exp(u).sum()
        p = torch.exp(u) / z
        lp = torch.log(torch.exp(u) / z) if none or bad else u - torch.log(z)
        ents.append(math.nan if bad else 0.0 if none else float(torch.log(z) - torch.where(p > 0, p * u, 0.0).sum()))
        lps.append(0.0 if i < 0 else -math.inf if i >= V or none else math.nan if bad else float(lp[i]))
        far.append(0.0 if not 0 <= i < V or none or bad or u[i] == -math.inf else abs(float(u[i])))
        order = []
        if n_top:
            sized, by = torch.sort(torch.where(torch.isnan(row), -math.inf, row), descending=True, stable=True)
            order = by[:n_top][sized[:n_top] > -math.inf].tolist()
        tops.append(order + [-1] * (n_top - len(order)))
        top_lps.append([math.nan if bad else float(lp[j]) for j in order] + [-math.inf] * (n_top - len(order)))
    d = lambda v: torch.tensor(v, dtype=torch.float64)
    return d(lps), d(ents), torch.tensor(tops).view(len(tops), -1), d(top_lps).view(len(tops), -1), d(far)


def near(got, want, bound, what):
    got = got.double().cpu()
    same = torch.isnan(got) & torch.isnan(want) | (got == want)
    off = torch.where(same, 0.0, (got - want).abs())
    assert bool((off <= bound).all()), f"{what}: {off.max()} off, {got.flatten()[off.argmax()]} for {want.flatten()[off.argmax()]}"


def compare(got, x, ids, n_top=0, temperature=None):
    lp, ent, top, top_lp, far = exact(x, ids, n_top, temperature)
    V = x.shape[1]
    unit = STEP * (V / 128 + 64)
    near(got[0], lp, unit * (1 + far + math.log(V)), "logprob")
    near(got[1], ent, 2 * unit * (1 + math.log(V)), "entropy")
    if n_top == 0:
        assert len(got) == 2 or got[2] is None and got[3] is None
        return
    assert got[2].dtype == torch.int32 and torch.equal(got[2].long().cpu(), top.long()), "alternatives"
    near(got[3], top_lp, unit * (1 + math.log(V) + torch.where(top_lp > -math.inf, top_lp.abs(), 0.0)), "alternatives' logprob")


def rows(n, V, dtype, seed, device, pad=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, V + pad, generator=g) * spread).to(dtype).to(device)
    ids = torch.randint(0, V, (n,), generator=g).to(device)
    t = (torch.rand(n, generator=g) * 1.5 + 0.2).to(device)
    return x[:, pad:], ids, t


DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,V,n_top,pad", [(1, 1, 1, 0), (3, 2, 2, 0), (5, 7, 3, 1), (2, 255, 20, 0), (4, 1000, 5, 3), (7, 4099, 1, 5),
                                           (2, 9001, 128, 1), (33, 2048, 0, 0), (1, 20011, 64, 7)])
def test_rows(device, dtype, n, V, n_top, pad):
    x, ids, t = rows(n, V, dtype, n * V, device, pad)
    compare(score.token_logprobs(x, ids, n_top), x, ids, n_top)
    compare(score.token_logprobs(x, ids, n_top, temperature=t), x, ids, n_top, t)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 9, 40, 150, 700, 2500])
def test_row_counts(n):
    """Few rows are split over several blocks, many are not: the same results either way."""
    x, ids, t = rows(n, 6007, torch.bfloat16, 3, "cuda", 3)
    got = score.token_logprobs(x, ids, 6, temperature=t)
    pick = sorted({0, n // 2, n - 1})
    at = torch.tensor(pick, device="cuda")
    compare(tuple(g[at] for g in got), x[at], ids[at], 6, t[at])
    one = score.token_logprobs(x[:1], ids[:1], 6, temperature=t[:1])
    assert torch.equal(one[2], got[2][:1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [1, 300])
def test_whole_vocabulary(dtype, n):
    x, ids, t = rows(n, 151936, dtype, 11, "cuda")
    got = score.token_logprobs(x, ids, 20, temperature=t)
    at = torch.tensor(sorted({0, n // 3, n - 1}), device="cuda")
    compare(tuple(g[at] for g in got), x[at], ids[at], 20, t[at])


def edge_rows(V, dtype):
    """Rows where a softmax goes wrong, and the token asked for in each."""
    low, inf = torch.finfo(dtype).min, math.inf
    g = torch.Generator().manual_seed(5)
    base = lambda: torch.randn(V, generator=g) * 2
    out = []

    def add(row, i):
        out.append((row.to(dtype), i))
    add(torch.full((V,), -inf), 1)                                    # a mask that leaves nothing
    r = torch.full((V,), -inf); r[V - 1] = 3.0; add(r, V - 1)         # ... and one token
    add(r.clone(), 0)                                                 # a masked token is asked for
    r = base(); r[: V // 2] = low; add(r, V - 1)                      # masks of the type's lowest value
    add(r.clone(), 0)
    add(torch.full((V,), low), V // 2)                                # nothing but those
    add(torch.zeros(V), V - 1)                                        # all tokens alike
    r = base(); r[V // 3] = math.nan; add(r, 0)
    r = base(); r[V // 3] = inf; add(r, V // 3)
    r = torch.full((V,), -inf); r[2] = math.nan; add(r, 2)
    r = base(); r[V // 2] = 90.0; add(r, V // 2)                      # certain
    add(r.clone(), 0)
    add(base(), -1)                                                   # nothing asked
    add(base(), V)                                                    # beyond the vocabulary
    add(base(), -(1 << 40))
    add(base() * 1e-30, 3)
    r = torch.zeros(V); r[1::2] = -0.0; add(r, 1)                     # zeros of both signs tie
    return torch.stack([r for r, _ in out]), torch.tensor([i for _, i in out])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,n_top", [(37, 5), (1500, 20), (6001, 3)])
@pytest.mark.parametrize("each", [True, False])
def test_edges(device, dtype, V, n_top, each):
    x, ids = edge_rows(V, dtype)
    x, ids = x.to(device), ids.to(device)
    if each:
        for r in range(x.shape[0]):
            compare(score.token_logprobs(x[r:r + 1], ids[r:r + 1], n_top), x[r:r + 1], ids[r:r + 1], n_top)
    else:
        compare(score.token_logprobs(x.repeat(40, 1), ids.repeat(40), n_top), x.repeat(40, 1), ids.repeat(40), n_top)
        t = torch.tensor([0.0, -1.0, 0.3, 2.0], device=device).repeat(x.shape[0])[:x.shape[0]]
        t = torch.where((x == torch.finfo(dtype).min).any(1), 1.0, t)     # (low - max) / T leaves the range of fp32 there
        compare(score.token_logprobs(x, ids, n_top, temperature=t), x, ids, n_top, t)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_candidates(device, dtype):
    """The largest scores side by side, and more ties than a list of candidates holds."""
    V = 40000
    g = torch.Generator().manual_seed(9)
    x = torch.randn(5, V, generator=g)
    x[0] = torch.arange(V).float() / 300                              # ascending
    x[1] = -torch.arange(V).float() / 300
    x[2, 5000:9000] = 4.5                                             # thousands of ties above everything
    x[3] = torch.where(torch.rand(V, generator=g) < 0.2, 3.0, -1.0)
    x[4] = torch.arange(V).float() % 8
    x, ids = x.to(dtype).to(device), torch.tensor([V - 1, 0, 7000, 3, 7]).to(device)
    for n_top in (1, 20, 128):
        compare(score.token_logprobs(x, ids, n_top), x, ids, n_top)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_scores_and_small_temperatures(device, dtype):
    """Scores of thousands, scores whose differences count in the 7th place, temperatures that leave one token, masks among them."""
    g = torch.Generator().manual_seed(21)
    V = 9000
    x = torch.randn(8, V, generator=g) * 3
    x[1] += 5000.0
    x[2] -= 30000.0
    x[3] *= 400.0
    x[4] = 1000.0 + torch.rand(V, generator=g)
    x[5, ::3] = -math.inf
    x[6, 100:] = -math.inf
    x[7, 50:8000] = torch.finfo(dtype).min
    x = x.to(dtype).to(device)
    ids = x.float().argmax(1)
    ids[::2] = 11
    compare(score.token_logprobs(x, ids, 3), x, ids, 3)
    for t in (1e-3, 1e-5, 1e-8, 30.0, 1e5):
        some = x[:7]
        T = torch.full((7,), t, device=device)
        compare(score.token_logprobs(some, ids[:7], 3, temperature=T), some, ids[:7], 3, T)


@pytest.mark.parametrize("device", DEVICES)
def test_strides_and_types(device):
    x, ids, t = rows(6, 500, torch.bfloat16, 2, device, 9)
    want = score.token_logprobs(x.contiguous(), ids, 4, temperature=t)
    wide = torch.zeros(12, dtype=torch.int64, device=device)
    wide[::2] = ids
    wide_t = torch.ones(18, device=device)
    wide_t[::3] = t
    # a row that starts elsewhere within 16 bytes is summed in another order, so not to the same bits: each is within the bound
    compare(want, x, ids, 4, t)
    compare(score.token_logprobs(x, wide[::2], 4, temperature=wide_t[::3]), x, ids, 4, t)
    every = x.contiguous().repeat_interleave(2, 0)
    compare(score.token_logprobs(every[::2], ids, 4, temperature=t), x, ids, 4, t)
    same = x[:1].expand(6, -1)                                        # rows of stride 0
    got = score.token_logprobs(same, ids, 2)
    compare(got, same, ids, 2)
    half = (torch.randn(3, 400, generator=torch.Generator().manual_seed(1)) * 2).half().to(device)
    compare(score.token_logprobs(half, ids[:3] % 400, 3), half, ids[:3] % 400, 3)


@pytest.mark.parametrize("device", DEVICES)
def test_no_rows(device):
    x = torch.empty(0, 50, device=device)
    ids = torch.empty(0, dtype=torch.int64, device=device)
    got = score.token_logprobs(x, ids, 3)
    assert [tuple(g.shape) for g in got] == [(0,), (0,), (0, 3), (0, 3)]
    h, w = torch.empty(0, 64, dtype=torch.bfloat16, device=device), torch.zeros(50, 64, dtype=torch.bfloat16, device=device)
    assert [tuple(g.shape) for g in score.head_logprobs(h, w, ids)] == [(0,), (0,)]


def test_refusals():
    x, ids = torch.zeros(4, 30), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError):
        score.token_logprobs(x, ids, 31)
    with pytest.raises(ValueError):
        score.token_logprobs(x, ids, -1)
    with pytest.raises(ValueError):
        score.token_logprobs(torch.zeros(2, 500), ids[:2], 129)
    with pytest.raises(ValueError):
        score.token_logprobs(x.T, torch.zeros(30, dtype=torch.int64))
    with pytest.raises(ValueError):
        score.token_logprobs(x[0], ids)
    with pytest.raises(ValueError):
        score.token_logprobs(x[:, :0], ids)
    with pytest.raises(TypeError):
        score.token_logprobs(x, ids.int())
    with pytest.raises(TypeError):
        score.token_logprobs(x.long(), ids)
    with pytest.raises(TypeError):
        score.token_logprobs(x, ids[:3])
    with pytest.raises(TypeError):
        score.token_logprobs(x, ids, temperature=torch.ones(3))
    with pytest.raises(TypeError):
        score.token_logprobs(x, ids, temperature=torch.ones(4, dtype=torch.float64))
    h, w = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(9, 16, dtype=torch.bfloat16)
    for bad in (w[:, :8], w.float(), w.T, w[:0], w[0]):
        with pytest.raises(ValueError):
            score.head_logprobs(h, bad, ids)
    with pytest.raises(ValueError):
        score.head_logprobs(h[:, :0], w[:, :0], ids)
    with pytest.raises(TypeError):
        score.head_logprobs(h, w, ids[:2])


def test_bounds_check(monkeypatch):
    from xllm_b200.ops._debug import BoundsError
    monkeypatch.setenv("XLLM_BOUNDS_CHECK", "1")
    x = torch.zeros(2, 30)
    score.token_logprobs(x, torch.tensor([-1, 29]))
    with pytest.raises(BoundsError):
        score.token_logprobs(x, torch.tensor([0, 30]))


@pytest.mark.gpu
def test_refusals_gpu():
    h, w = torch.zeros(4, 20, dtype=torch.bfloat16, device="cuda"), torch.zeros(9, 20, dtype=torch.bfloat16, device="cuda")
    ids = torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError):
        score.head_logprobs(h, w, ids)                                # a width that is no multiple of 8
    with pytest.raises(ValueError):
        score.head_logprobs(h[:, 1:17], w[:, 1:17], ids)              # rows off the 16-byte boundaries
    with pytest.raises(ValueError):
        score.head_logprobs(h[:, :16].float(), w[:, :16].float(), ids)
    with pytest.raises(TypeError):
        score.token_logprobs(h, ids.cpu())
    with pytest.raises(ValueError):
        score.head_logprobs(h[:, :16].contiguous(), w[:, :16].contiguous().cpu(), ids)


def test_too_many_rows():
    """More than a kernel counts in 32 bits, of one row in memory."""
    n = 2 ** 32 + 5
    x, ids = torch.zeros(1, 8, dtype=torch.bfloat16).expand(n, -1), torch.zeros(1, dtype=torch.int64).expand(n)
    with pytest.raises(ValueError):
        score.token_logprobs(x, ids)
    with pytest.raises(ValueError):
        score.head_logprobs(x, x[:3], ids)


@pytest.mark.parametrize("columns", [(1 << 30) + 1, (1 << 31) - 1, (1 << 32) + 5])
def test_too_many_columns(columns):
    """More than a kernel counts in 32 bits; nothing of them is read."""
    e = lambda *shape, dtype=torch.bfloat16: torch.empty(*shape, dtype=dtype, device="meta")
    ids = e(1, dtype=torch.int64)
    with pytest.raises(ValueError, match="columns"):
        score.token_logprobs(e(1, columns), ids)
    with pytest.raises(ValueError, match="columns"):
        score.head_logprobs(e(1, columns), e(3, columns), ids)
    with pytest.raises(ValueError, match="vocabulary"):
        score.head_logprobs(e(1, 8), e(columns, 8), ids)


# ------------------------------------------------------------------------------- from hidden states
def head_case(T, K, V, seed, device, spread=1.4):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, K, generator=g) * spread / math.sqrt(K)).to(torch.bfloat16)
    ids = torch.randint(0, V, (T,), generator=g)
    h = (torch.randn(T, K, generator=g) + torch.rand(T, 1, generator=g) * 3 * w[ids].float()).to(torch.bfloat16)
    t = torch.rand(T, generator=g) * 1.5 + 0.3
    return h.to(device), w.to(device), ids.to(device), t.to(device)


def compare_head(got, h, w, ids, temperature=None):
    """A score is a sum of K exact products: off by at most 2^-23 of the sum of their sizes an addition, truncated.  A
    log-probability moves by at most twice as much as the scores, the entropy H by at most 2 H times."""
    x = h.double().cpu() @ w.double().cpu().T
    size = (h.double().cpu().abs() @ w.double().cpu().abs().T).amax(1)
    T = torch.ones(len(x)).double() if temperature is None else temperature.double().cpu()
    off = h.shape[1] * 2.0 ** -23 * size / torch.where(T > 0, T, 1.0)
    lp, ent, _, _, far = exact(x, ids, 0, temperature)
    V = w.shape[0]
    unit = STEP * (V / 128 + 64)
    near(got[0], lp, 2 * off + unit * (1 + far + math.log(V)), "logprob")
    near(got[1], ent, (2 * off + 2 * unit) * (1 + math.log(V)), "entropy")
    assert got[0].dtype == got[1].dtype == torch.float32


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T,K,V", [(1, 8, 1), (1, 64, 17), (3, 72, 300), (5, 200, 513), (64, 64, 255), (129, 136, 256), (257, 64, 1031),
                                   (2, 1000, 4099)])
def test_head(device, T, K, V):
    h, w, ids, t = head_case(T, K, V, T + K + V, device)
    compare_head(score.head_logprobs(h, w, ids), h, w, ids)
    compare_head(score.head_logprobs(h, w, ids, temperature=t), h, w, ids, t)


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,V", [(1, 4096, 151936), (16, 512, 50257), (17, 264, 30000), (63, 512, 20000), (65, 512, 20000), (32, 2048, 32000), (45, 1024, 129280), (100, 512, 32003), (130, 512, 32768),
                                   (300, 2880, 9000), (1000, 256, 40000), (4097, 128, 12345), (129, 2048, 3001), (200, 1024, 20000), (256, 1208, 5000)])
def test_head_sizes(T, K, V):
    h, w, ids, t = head_case(T, K, V, 7, "cuda")
    got = score.head_logprobs(h, w, ids, temperature=t)
    at = torch.tensor(sorted({0, T // 2, T // 3, T - 1}), device="cuda")
    compare_head(tuple(g[at] for g in got), h[at], w, ids[at], t[at])
    assert score.error_status() == 0


@pytest.mark.parametrize("device", DEVICES)
def test_head_edges(device):
    h, w, ids, t = head_case(12, 64, 700, 3, device)
    ids[0], ids[1], ids[2] = -1, 700, 699
    t[3], t[4] = 0.0, -2.0
    h[5] = 0                                                          # every score alike
    h[6] *= 40                                                        # one token certain
    compare_head(score.head_logprobs(h, w, ids, temperature=t), h, w, ids, t)
    h[7, 3], h[8, 5] = math.nan, math.inf
    w[11, 5] = w[:, 5].abs().max()                                    # a positive weight: some score is +inf
    got = score.head_logprobs(h, w, ids)
    assert torch.isnan(got[0][7:9]).all() and torch.isnan(got[1][7:9]).all()
    keep = torch.tensor([i for i in range(12) if i not in (7, 8)], device=device)
    compare_head(tuple(g[keep] for g in got), h[keep], w, ids[keep])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T,K,V", [(40, 512, 3000), (150, 1000, 3000)])
@pytest.mark.parametrize("low", [1e-5, 1e-7, 1e-9, 1e-30])
def test_head_lowest_temperatures(device, T, K, V, low):
    """A token ahead of all others by 0.01 is certain at temperatures that magnify the sums' own rounding to more than the others are
    behind.  What is left is the rounding of a term of up to 2^1 taken out of its own logarithm: an exponential, a sum, a
    logarithm, a quotient and a product, 2^-22 each at most."""
    h, w, _, _ = head_case(T, K, V, 11, device)
    best = (h.double().cpu() @ w.double().cpu().T).topk(2)
    sure = best.values[:, 0] - best.values[:, 1] > 0.01
    assert sure.sum() > T // 2
    lp, ent = score.head_logprobs(h, w, best.indices[:, 0].to(device), temperature=torch.full((T,), low, device=device))
    assert lp.cpu()[sure].abs().max() <= 2.0 ** -19 and ent.cpu()[sure].abs().max() <= 2.0 ** -19


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("low", [1e-30, 5e-39, 2e-39, 1e-44])
def test_temperatures_without_an_inverse(device, low):
    """The inverse of what fp32 holds below 2.9e-39 is beyond fp32: the most likely token is certain all the same, the others never occur,
    and of two alike each has half."""
    x = torch.tensor([[3.0, -1.0, 2.0, -math.inf, 0.5], [1.0, 4.0, 4.0, 0.0, -8.0]]).repeat(2, 1).to(device)
    ids = torch.tensor([0, 1, 2, 3], device=device)
    t = torch.full((4,), low, device=device)
    lp, ent, top, top_lp = score.token_logprobs(x, ids, 2, temperature=t)
    half = math.log(0.5)
    near(lp[:2], torch.tensor([0.0, half]), 2.0 ** -20, "logprob")                # a logarithm and its sum
    assert (lp[2:] < -1e29).all() and top.tolist() == [[0, 2], [1, 2]] * 2
    near(ent, torch.tensor([0.0, -half] * 2), 2.0 ** -20, "entropy")
    near(top_lp[:, 0], torch.tensor([0.0, half] * 2), 2.0 ** -20, "alternatives")
    h = torch.eye(16, dtype=torch.bfloat16, device=device)[:4]
    w = torch.zeros(5, 16, dtype=torch.bfloat16, device=device)
    w[:, :4] = torch.where(x == -math.inf, -50.0, x).T.to(torch.bfloat16)
    lp, ent = score.head_logprobs(h, w, ids, temperature=t)
    near(lp[:2], torch.tensor([0.0, half]), 2.0 ** -20, "logprob")
    assert (lp[2:] < -1e29).all()
    near(ent, torch.tensor([0.0, -half] * 2), 2.0 ** -20, "entropy")


@pytest.mark.parametrize("device", DEVICES)
def test_head_strides(device):
    h, w, ids, t = head_case(9, 128, 333, 4, device)
    want = score.head_logprobs(h, w, ids, temperature=t)
    wide_h, wide_w = torch.full((9, 200), math.nan, dtype=h.dtype, device=device), torch.full((400, 136), math.nan, dtype=h.dtype, device=device)
    wide_h[:, 8:136], wide_w[:333, :128] = h, w
    for a, b in zip(want, score.head_logprobs(wide_h[:, 8:136], wide_w[:333, :128], ids, temperature=t)):
        assert torch.equal(a, b)
    same = h[:1].expand(9, -1)
    compare_head(score.head_logprobs(same, w, ids), same, w, ids)


@pytest.mark.gpu
def test_bits_repeat_and_streams():
    """The same call gives the same bits, on a stream of its own too, and beside another one."""
    x, ids, t = rows(5, 30000, torch.bfloat16, 8, "cuda")
    h, w, hid, ht = head_case(70, 256, 20000, 8, "cuda")
    a, b = score.token_logprobs(x, ids, 9, temperature=t), score.head_logprobs(h, w, hid, temperature=ht)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append((score.token_logprobs(x, ids, 9, temperature=t), score.head_logprobs(h, w, hid, temperature=ht)))
    torch.cuda.synchronize()
    for c, d in got:
        assert all(torch.equal(p, q) for p, q in zip(a, c)) and all(torch.equal(p, q) for p, q in zip(b, d))


@pytest.mark.gpu
def test_captured():
    """Two graphs, replayed after each other with other inputs in the same places."""
    from xllm_b200.ops import gemm_tcgen05
    gemm_tcgen05.prepare()
    x, ids, t = rows(40, 5000, torch.bfloat16, 8, "cuda")
    h, w, hid, ht = head_case(33, 128, 3000, 9, "cuda")
    call = [lambda: score.token_logprobs(x, ids, 5, temperature=t), lambda: score.head_logprobs(h, w, hid, temperature=ht)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for f in call:
            f()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for f in call + call:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = f()
        graphs.append((g, out, f))
    x2, ids2, _ = rows(40, 5000, torch.bfloat16, 18, "cuda")
    h2, _, hid2, _ = head_case(33, 128, 3000, 19, "cuda")
    x.copy_(x2), ids.copy_(ids2), h.copy_(h2), hid.copy_(hid2)
    for g, _, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    for _, out, f in graphs:
        for a, b in zip(out, f()):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_captured_first_calls():
    """A process whose first calls are captured ones."""
    import subprocess
    import sys
    code = """
import torch
from xllm_b200.ops import score, tables
x, ids = torch.randn(9, 3000, device="cuda").bfloat16(), torch.arange(9, device="cuda")
h, w = torch.randn(9, 64, device="cuda").bfloat16(), torch.randn(3000, 64, device="cuda").bfloat16()
many = torch.randn(300, 64, device="cuda").bfloat16()
i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
table, ctx, new, free = torch.zeros(2, 4, dtype=torch.int32, device="cuda"), i32(3, 0), i32(2, 5), i32(7, 8, 9)
calls = [lambda: score.token_logprobs(x, ids, 4), lambda: score.head_logprobs(h, w, ids),
         lambda: score.head_logprobs(many, w, ids.repeat(34)[:300]), lambda: tables.step_tables(table, ctx, new, 4, 9, free)]
torch.cuda.synchronize()
graphs = []
for f in calls:
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = f()
    graphs.append((g, out))
for g, _ in graphs:
    g.replay()
torch.cuda.synchronize()
for (_, out), f in zip(graphs, calls):
    assert all(torch.equal(a, b) for a, b in zip(out, f()))
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


@pytest.mark.gpu
def test_rows_beyond_32_bits():
    """Row offsets that pass 2^31 elements."""
    V = 151936
    n = (1 << 31) // V + 3
    x = torch.zeros(n, V, dtype=torch.bfloat16, device="cuda")
    y, ids, _ = rows(3, V, torch.bfloat16, 6, "cuda")
    x[-3:] = y
    every = torch.zeros(n, dtype=torch.int64, device="cuda")
    every[-3:] = ids
    got = score.token_logprobs(x, every, 2)
    compare(tuple(g[-3:] for g in got), y, ids, 2)
    assert abs(float(got[0][0]) + math.log(V)) < 1e-4 and got[2][0].tolist() == [0, 1]


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,V", [(40, 4096, 8192), (300, 4096, 8192), (300, 2048, 8192)])
def test_head_cut_sums(T, K, V):
    """What the tensor cores cut off a sum of K products is 0.94e-9 K of it on average, with an error half as large for scores of random signs
    (0.83 to 1.00e-9).  Made up for, the results are off by at most a quarter of what scores shorter by that would be off, and the
    roundings of a log-probability, 8 of 2^-24."""
    h, w, ids, t = head_case(T, K, V, 13, "cuda", spread=2.0)
    x = h.double() @ w.double().T
    cut = 0.94e-9 * K

    def results(x):
        lp = torch.log_softmax(x, dim=1)
        return lp.gather(1, ids[:, None])[:, 0], -(lp.exp() * lp).sum(1)
    for got, want, short in zip(score.head_logprobs(h, w, ids), results(x), results(x * (1 - cut))):
        off, without = (got.double() - want).norm(), (short - want).norm()
        assert float(off) <= 0.25 * float(without) + 8 * STEP * float(want.norm()), (float(off), float(without))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T,K,V", [(64, 512, 3000), (100, 64, 700), (300, 1000, 3000)])
def test_head_signs(device, T, K, V):
    """A log-probability is not above 0 and an entropy not below, to the last bit: with tokens that are certain, nearly so, and others."""
    h, w, ids, t = head_case(T, K, V, 17, device)
    h = (h.float() + torch.linspace(0, 40, T, device=device)[:, None] * w[ids].float()).to(torch.bfloat16)
    for temperature in (None, t, t * 1e-3):
        lp, ent = score.head_logprobs(h, w, ids, temperature=temperature)
        assert bool((lp <= 0).all()) and bool((ent >= 0).all()), (float(lp.max()), float(ent.min()))


def sums_case(kind, T, K, V, device):
    """Hidden states whose scores' partial sums do not grow evenly over K."""
    g = torch.Generator().manual_seed(K + T)
    w = (torch.randn(V, K, generator=g)).to(torch.bfloat16)
    h = torch.zeros(T, K)
    if kind == "one":                                                 # one channel other than 0
        h[torch.arange(T), torch.randint(0, K, (T,), generator=g)] = 6.0
    elif kind == "few":
        for r in range(T):
            h[r, torch.randperm(K, generator=g)[:4]] = 3.0
    elif kind in ("first", "last"):                                   # one channel far larger than all others
        h = torch.randn(T, K, generator=g) * 0.1 / math.sqrt(K)
        h[:, 0 if kind == "first" else K - 1] = 6.0
    elif kind == "cancel":                                            # the second half takes back most of the first one
        h = torch.randn(T, K, generator=g) * 12 / math.sqrt(K)
        h[:, K // 2:] = -h[:, :K // 2]
        w[:, K // 2:] = (w[:, :K // 2].float() + 0.3 * torch.randn(V, K // 2, generator=g)).to(torch.bfloat16)
    ids = torch.randint(0, V, (T,), generator=g)
    return h.to(torch.bfloat16).to(device), w.to(device), ids.to(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["one", "few", "first", "last", "cancel"])
@pytest.mark.parametrize("T,K,V", [(40, 4096, 2000), (150, 4096, 1000), (40, 1536, 2000)])
def test_head_uneven_sums(device, kind, T, K, V):
    """Whatever order a score's products come in: no more than 1024 of them are summed in the tensor cores, in 64 steps, each of which cuts
    off less than 2^-23 of the largest partial sum and half of that on average, so together 64 of 2^-24 of it; and next to nothing
    of a sum of few products.  A log-probability moves by at most as much as the scores, and has 8 roundings to fp32 of its own."""
    h, w, ids = sums_case(kind, T, K, V, device)
    x, partial = torch.zeros(T, V, dtype=torch.float64), torch.zeros(T, dtype=torch.float64)
    hd, wd = h.double().cpu(), w.double().cpu()
    for k in range(0, K, 64):
        x += hd[:, k:k + 64] @ wd[:, k:k + 64].T
        partial = torch.maximum(partial, x.abs().amax(1))
    lp = torch.log_softmax(x, dim=1)
    want = lp.gather(1, ids.cpu()[:, None])[:, 0], -(lp.exp() * lp).sum(1)
    got = score.head_logprobs(h, w, ids)
    cut = 0.0 if kind in ("one", "few") else 64 * STEP * float(partial.norm())
    for a, b, name in zip(got, want, ("logprob", "entropy")):
        off = float((a.double().cpu() - b).norm())
        assert off <= cut + 8 * STEP * float(torch.stack(want).abs().amax(0).norm()), (name, off, cut, float(b.norm()))


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,V", [(1, 1024, 70000), (1, 2056, 40000), (8, 1032, 9000), (63, 1040, 66000), (64, 1104, 65000), (65, 1104, 65000),
                                   (100, 704, 100000), (127, 2880, 30000), (128, 512, 20011), (128, 1000, 70000), (128, 4104, 17000),
                                   (129, 1032, 5003), (130, 1792, 3000), (256, 1800, 4111), (257, 904, 6000), (1000, 2048, 3333),
                                   (4097, 128, 12345), (4100, 1088, 2051)])
def test_head_every_row(T, K, V):
    """Every row, around the numbers of rows and products where the kernel takes another form.  A score is off by what at most 64 steps
    of the tensor cores cut off, less than 2^-23 of the sum of its products' sizes each, and by a rounding for every chunk of 896 products
    that is added; a log-probability moves by at most twice as much and has the roundings of `compare`."""
    h, w, ids, t = head_case(T, K, V, 23, "cuda")
    ids[::5] = -1
    for temperature in (None, t):
        T0 = torch.ones(T, device="cuda").double() if temperature is None else temperature.double()
        u = h.double() @ w.double().T / T0[:, None]
        size = (h.double().abs() @ w.double().abs().T).amax(1) / T0
        lp = torch.log_softmax(u, dim=1)
        off = 2 * size * (min(K / 16, 64) * 2.0 ** -23 + (K / 896 + 1) * STEP)
        unit = STEP * (V / 128 + 64)
        got = score.head_logprobs(h, w, ids, temperature=temperature)
        asked = lp.gather(1, ids.clamp(min=0)[:, None])[:, 0]
        far = torch.where(ids < 0, 0.0, (u.amax(1) - u.gather(1, ids.clamp(min=0)[:, None])[:, 0]))
        near(got[0], torch.where(ids < 0, 0.0, asked).cpu(), (off + unit * (1 + far + math.log(V))).cpu(), "logprob")
        near(got[1], -(lp.exp() * lp).sum(1).cpu(), ((off + 2 * unit) * (1 + math.log(V))).cpu(), "entropy")
    assert score.error_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,V", [(33, 2056, 9000), (100, 1032, 9000), (300, 2056, 9000)])
def test_chunked_rows_repeat(T, K, V):
    """Sums of several chunks have the same bits in every call: beside another call on another stream, and captured, where the replayed
    graph reads what is in its inputs' places then."""
    from xllm_b200.ops import gemm_tcgen05
    gemm_tcgen05.prepare()
    h, w, ids, t = head_case(T, K, V, 31, "cuda")
    h2, _, ids2, _ = head_case(T, K, V, 32, "cuda")
    want, want2 = score.head_logprobs(h, w, ids, temperature=t), score.head_logprobs(h2, w, ids2, temperature=t)
    torch.cuda.synchronize()
    got, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for _ in range(6):
        for s, a, b in zip(streams, (h, h2), (ids, ids2)):
            with torch.cuda.stream(s):
                got.append(score.head_logprobs(a, w, b, temperature=t))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(out, (want, want2)[i % 2]))
    g, place, asked = torch.cuda.CUDAGraph(), h.clone(), ids.clone()
    with torch.cuda.graph(g):
        out = score.head_logprobs(place, w, asked, temperature=t)
    for a, b, c in ((h, ids, want), (h2, ids2, want2), (h, ids, want)):
        place.copy_(a), asked.copy_(b)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, c))
    assert score.error_status() == 0

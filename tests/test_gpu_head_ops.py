"""The model-side operators (flashtrie_device.adapter_logits, propose,
sequence_logp, preference_loss, bs_tbs_hidden) against plain 64-bit
implementations.

Tolerances, derived here once (u = 2^-24, half a step of f32):
  - a softmax sum: each exponential's argument (x - m) log2(e) is off by two
    roundings, at most 2 u S with S the spread of the row's finite logits, the
    base-2 exponential by 2 steps (4 u), and a thread adds at most V/32 + 64
    values in sequence.  REL_Z = (4 S + 4 + V/32 + 64) u bounds its relative
    error, and so the absolute error of a log-sum;
  - a matrix product of inner length D summed in 32 bits in any order:
    2 D u sum|a b| (two roundings a step, which covers truncation too);
  - a result rounded to type t: half of finfo(t).eps relative, or half the
    smallest subnormal.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
FLT_MAX = 3.4028234663852886e38
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALVES = [torch.bfloat16, torch.float16]
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


@pytest.fixture(scope="module")
def fd(built):
    import flashtrie_device
    return flashtrie_device


def dev():
    return torch.device("cuda:0")


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def half_step(t, ref):
    return torch.finfo(t).eps / 2 * ref.abs() + TINY[t]


def spread(x):
    """Largest difference of finite logits in a row (0 for empty rows)."""
    f = torch.isfinite(x)
    hi = torch.where(f, x, -math.inf).amax(-1)
    lo = torch.where(f, x, math.inf).amin(-1)
    return torch.where(hi >= lo, hi - lo, 0.0).clamp(min=0)


def rel_z(x):
    return (4 * spread(x) + 4 + x.shape[-1] / 32 + 64) * U


def make_logits(n, L, V, t, seed, masked=True):
    g = gen(seed)
    x = torch.randn((n, L, V), generator=g, device="cuda") * 2
    if masked and V > 3:
        x[torch.rand((n, L, V), generator=g, device="cuda") < 0.1] = -math.inf
    return x.to(t)


# ------------------------------------------------------------------ propose

def propose_oracle(x, k, order):
    x = x.double().cpu()
    n, L, V = x.shape
    ids = torch.full((n, L, k), -1, dtype=torch.int64)
    lps = torch.full((n, L, k), -FLT_MAX, dtype=torch.float64)
    for i in range(n):
        for l in range(L):
            row = x[i, l]
            if torch.isnan(row).any() or (row == math.inf).any() or (row == -math.inf).all():
                continue
            lp = torch.log_softmax(row, 0)
            at = torch.argsort(row, descending=True, stable=True)
            at = at[row[at] > -math.inf][:k]
            if order == "id":
                at = torch.sort(at).values
            ids[i, l, :at.numel()] = at
            lps[i, l, :at.numel()] = lp[at]
    return ids, lps


def check_propose(fd, x, k, order):
    ids, lps = fd.propose(x, k, order=order)
    want_ids, want = propose_oracle(x, k, order)
    assert ids.dtype == torch.int32 and lps.dtype == torch.float32 and ids.shape == want_ids.shape
    assert torch.equal(ids.cpu().long(), want_ids)
    pad = want_ids < 0
    assert bool((lps.cpu()[pad] == -FLT_MAX).all())
    xd = x.double().cpu()
    # x - m and the result are rounded once each, the logarithm of the sum by
    # two steps (of a value below log V + 1) beside the sum's own error.
    tol = (rel_z(xd) + 4 * U * (math.log(xd.shape[-1]) + 1))[..., None] + 2 * U * torch.where(pad, 0.0, want).abs()
    tol = tol + U * spread(xd)[..., None]
    err = torch.where(pad, 0.0, (lps.cpu().double() - want).abs())
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,L,V,k", [(1, 1, 1, 1), (1, 1, 1, 3), (2, 3, 5, 5), (1, 2, 7, 8192), (3, 1, 31, 4),
                                     (2, 2, 4099, 64), (1, 3, 32000, 1000), (2, 1, 9001, 8192), (1, 2, 100003, 1000),
                                     (40, 5, 1021, 100), (1, 1, 300001, 2000)])
def test_propose_matches_oracle(fd, t, n, L, V, k):
    x = make_logits(n, L, V, t, seed=V + k)
    check_propose(fd, x, k, "id")
    check_propose(fd, x, k, "logp")


@pytest.mark.parametrize("t", TYPES)
def test_propose_ties_go_to_the_lowest_ids(fd, t):
    V = 70001
    x = torch.zeros((1, 4, V), device="cuda")
    x[0, 1, ::2] = -0.0  # equal to 0
    x[0, 2] = (torch.arange(V, device="cuda") % 7).float()
    x[0, 3, V - 5:] = 1.0
    for k in (1, 100, 5000):
        check_propose(fd, x.to(t), k, "id")
        check_propose(fd, x.to(t), k, "logp")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rising", [True, False])
def test_propose_sorted_logits(fd, t, rising):
    """Logits that rise or fall with the id: every later value beats all
    before it, or none does."""
    V = 150001
    x = torch.linspace(-20, 20, V, device="cuda")
    x = (x if rising else x.flip(0)).expand(1, 2, V).contiguous().to(t)
    check_propose(fd, x, 1000, "id")
    check_propose(fd, x, 8192, "logp")


@pytest.mark.parametrize("t", TYPES)
def test_propose_best_in_one_place(fd, t):
    """All of the best logits within one stretch, at the row's end, its start
    or its middle."""
    V, k = 200003, 1500
    x = torch.randn((1, 3, V), generator=gen(1), device="cuda").clamp(max=4.0)
    for l, at in enumerate((V - k, 0, V // 2)):
        x[0, l, at:at + k] = 6 + torch.arange(k, device="cuda") * 0.001
    check_propose(fd, x.to(t), k, "id")


@pytest.mark.parametrize("t", TYPES)
def test_propose_empty_and_broken_rows(fd, t):
    V = 12345
    x = make_logits(1, 6, V, t, seed=5)
    x[0, 0] = -math.inf
    x[0, 1, 77] = math.nan
    x[0, 2, 99] = math.inf
    x[0, 3] = -math.inf
    x[0, 3, V - 1] = -3.0
    x[0, 4] = torch.finfo(t).min
    check_propose(fd, x, 50, "id")
    check_propose(fd, x, 50, "logp")


def test_propose_unaligned_rows_leave_neighbours_alone(fd):
    """A contiguous view that starts in the middle of a vector, and outputs
    that are written whole."""
    base = torch.randn(5 + 3 * 1001, generator=gen(9), device="cuda")
    for t in TYPES:
        b = base.to(t)
        b[:5] = math.nan
        check_propose(fd, b[5:].view(1, 3, 1001), 40, "logp")


def test_propose_all_equal(fd):
    """Every logit passes any bound: the lowest ids win."""
    x = torch.full((1, 2, 300001), 1.5, device="cuda")
    for t in TYPES:
        for k in (1, 1000, 8192):
            check_propose(fd, x.to(t), k, "id")


def test_propose_mostly_zeros(fd):
    """The bound falls on a logit of 0, which thousands share, in rows of
    several stretches."""
    x = torch.relu(torch.randn((1, 3, 300001), generator=gen(8), device="cuda") - 3)
    x[0, 1] = torch.where(x[0, 1] > 0, x[0, 1], -0.0)
    x[0, 2, 5:] = torch.where(x[0, 2, 5:] > 0, x[0, 2, 5:], -1e-30)
    for t in (torch.float32, torch.bfloat16):
        for k in (300, 1000, 6000):
            check_propose(fd, x.to(t), k, "id")


def test_propose_few_bounds_hold(fd):
    """Rows whose best logits the sample sees too often or not at all."""
    V = 262144
    x = torch.randn((1, 4, V), generator=gen(3), device="cuda")
    where = torch.arange(V, device="cuda")
    x[0, 0, where % 128 < 16] += 9  # stretches of 16
    x[0, 1, (where + 64) % 128 < 16] += 9
    x[0, 2, :700] += 9
    x[0, 3, where % 131 == 5] += 9
    for t in TYPES:
        check_propose(fd, x.to(t), 1200, "logp")


def test_propose_beyond_2_31_entries(fd):
    V, rows = 2200000, 1000
    x = torch.empty((1, rows, V), dtype=torch.bfloat16, device="cuda").fill_(-4.0)
    for l in (0, 976, 999):
        x[0, l] = torch.randn(V, generator=gen(l), device="cuda").to(torch.bfloat16)
    ids, lps = fd.propose(x, 100)
    for l in (0, 976, 999):
        want_ids, want = propose_oracle(x[:, l:l + 1], 100, "id")
        assert torch.equal(ids[:, l:l + 1].cpu().long(), want_ids)
    assert torch.equal(ids[0, 500].cpu().long(), torch.arange(100))


def test_propose_no_rows(fd):
    ids, lps = fd.propose(torch.empty((0, 4, 10), device="cuda"), 3)
    assert ids.shape == lps.shape == (0, 4, 3)


# ------------------------------------------------------------ adapter_logits

def make_head(n, L, V, D, r, G, t, seed):
    g = gen(seed)
    h = torch.randn((n, L, D), generator=g, device="cuda").to(t)
    w = (torch.randn((V, D), generator=g, device="cuda") / math.sqrt(D)).to(t)
    a = (torch.randn((G, r, D), generator=g, device="cuda") / math.sqrt(D)).to(t)
    b = (torch.randn((G, V, r), generator=g, device="cuda") * 0.3).to(t)
    s = torch.rand(G, generator=g, device="cuda") + 0.5
    ids = torch.randint(-1, G, (n,), generator=g, device="cuda", dtype=torch.int32)
    return h, w, ids, a, b, s


def adapter_oracle(h, w, ids=None, a=None, b=None, s=None):
    """(logits, sum of the absolute products) in 64 bits."""
    h, w = h.double(), w.double()
    y, m = h @ w.T, h.abs() @ w.abs().T
    for i, at in enumerate(ids.tolist() if ids is not None else []):
        if at == -1:
            continue
        if not 0 <= at < a.shape[0]:
            y[i] = math.nan
            continue
        f = float(s[at]) if s is not None else 1.0
        y[i] += f * ((h[i] @ a[at].double().T) @ b[at].double().T)
        m[i] += abs(f) * ((h[i].abs() @ a[at].double().abs().T) @ b[at].double().abs().T)
    return y, m


def check_adapter(out, y, m, D, r, t):
    """The low-rank values lose 2^-17 (two bf16 parts: what the first leaves is
    at most 2^-8 of its power of two, a value of the power 2^-9 or below, of
    which the second leaves 2^-8) or less beside the 32-bit sums; the result is
    rounded once."""
    tol = (2 * (D + 4 * r + 8) * U + 2.0 ** -17) * m + half_step(out.dtype, y)
    bad = torch.isnan(y)
    assert bool((torch.isnan(out) == bad).all())
    err = torch.where(bad, 0.0, (out.double() - y).abs())
    tol = torch.where(bad, 0.0, tol)
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("n,L,V,D,r,G", [(1, 1, 1, 8, 8, 1), (1, 1, 127, 64, 8, 1), (3, 5, 129, 72, 16, 2),
                                         (2, 20, 1000, 256, 64, 3), (5, 1, 4097, 200, 24, 9), (70, 1, 333, 136, 16, 90),
                                         (9, 33, 777, 64, 8, 2), (1, 300, 515, 320, 128, 1), (17, 16, 260, 1032, 40, 4),
                                         (6, 50, 640, 128, 256, 4), (300, 2, 256, 64, 32, 5)])
def test_adapter_logits_match_oracle(fd, t, n, L, V, D, r, G):
    h, w, ids, a, b, s = make_head(n, L, V, D, r, G, t, seed=n + V + D)
    y, m = adapter_oracle(h, w, ids, a, b, s)
    for out_t in (t, torch.float32):
        out = fd.adapter_logits(h, w, ids, a, b, s, out_dtype=out_t)
        assert out.dtype == out_t and out.shape == (n, L, V)
        check_adapter(out, y, m, D, r, t)


@pytest.mark.parametrize("t", HALVES)
def test_adapter_logits_without_adapters_or_scale(fd, t):
    h, w, ids, a, b, s = make_head(4, 3, 500, 96, 8, 2, t, seed=3)
    y, m = adapter_oracle(h, w)
    check_adapter(fd.adapter_logits(h, w), y, m, 96, 0, t)
    none = torch.full_like(ids, -1)
    check_adapter(fd.adapter_logits(h, w, none, a, b, s), y, m, 96, 8, t)
    y, m = adapter_oracle(h, w, ids, a, b)
    check_adapter(fd.adapter_logits(h, w, ids, a, b), y, m, 96, 8, t)


@pytest.mark.parametrize("t", HALVES)
def test_adapter_ids_out_of_range_are_nan(fd, t):
    """Only the request that names the wrong adapter is NaN."""
    h, w, ids, a, b, s = make_head(6, 7, 300, 64, 16, 3, t, seed=4)
    ids = torch.tensor([0, 3, -1, -2, 2, 2147483647], dtype=torch.int32, device="cuda")
    y, m = adapter_oracle(h, w, ids, a, b, s)
    out = fd.adapter_logits(h, w, ids, a, b, s)
    assert bool(torch.isnan(out[[1, 3, 5]]).all()) and not bool(torch.isnan(out[[0, 2, 4]]).any())
    check_adapter(out, y, m, 64, 16, t)


@pytest.mark.parametrize("t", HALVES)
def test_adapter_logits_nan_stays_in_its_request(fd, t):
    """An infinity in one request's hidden state, or in an adapter that one
    request uses, reaches no other request."""
    h, w, ids, a, b, s = make_head(5, 4, 257, 128, 8, 3, t, seed=5)
    ids = torch.tensor([0, 1, 2, 0, -1], dtype=torch.int32, device="cuda")
    h[3, 2, 5] = math.inf
    a[1, 3, 7] = math.nan
    out = fd.adapter_logits(h, w, ids, a, b, s)
    clean = torch.ones((5, 4), dtype=torch.bool, device="cuda")
    clean[1] = False
    clean[3, 2] = False
    y, m = adapter_oracle(h, w, ids, a, b, s)
    check_adapter(out[clean], y[clean], m[clean], 128, 8, t)
    assert not bool(torch.isfinite(out[1]).any())


def test_adapter_logits_same_bits_every_time(fd):
    h, w, ids, a, b, s = make_head(33, 20, 5000, 512, 16, 6, torch.bfloat16, seed=6)
    first = fd.adapter_logits(h, w, ids, a, b, s, out_dtype=torch.float32)
    for _ in range(3):
        assert torch.equal(first, fd.adapter_logits(h, w, ids, a, b, s, out_dtype=torch.float32))
    assert fd.adapter_logits(h[:0], w, ids[:0], a, b, s).shape == (0, 20, 5000)


@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("n,L,V,D,r,G", [(1, 300, 80001, 72, 64, 1), (1, 1, 80000, 64, 8, 2), (20, 20, 76000, 136, 40, 6),
                                         (3, 40, 90001, 1096, 16, 2), (2, 30, 76032, 1160, 72, 3),
                                         (5, 60, 1001, 1032, 24, 2), (300, 1, 1000, 64, 8, 290), (9000, 1, 130, 16, 8, 3)])
def test_adapter_logits_wide_and_long(fd, t, n, L, V, D, r, G):
    """Vocabularies and batches that take two halves to a tile, several tiles
    of tokens, long inner dimensions, slices of the low-rank dimension, groups
    wider than a stage, and more requests than are sorted."""
    h, w, ids, a, b, s = make_head(n, L, V, D, r, G, t, seed=n + V + D)
    y, m = adapter_oracle(h, w, ids, a, b, s)
    for out_t in (t, torch.float32):
        check_adapter(fd.adapter_logits(h, w, ids, a, b, s, out_dtype=out_t), y, m, D, r, t)
    y, m = adapter_oracle(h, w)
    check_adapter(fd.adapter_logits(h, w, out_dtype=torch.float32), y, m, D, 0, t)


@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("n,L,G", [(6, 20, 3), (6, 1, 6), (1, 5, 2)])
def test_adapter_infinities_stay_with_their_requests(fd, t, n, L, G):
    """An adapter whose B holds infinities and NaN reaches the requests that
    use it, at those vocabulary entries, and nothing else."""
    h, w, ids, a, b, s = make_head(n, L, 400, 64, 16, G, t, seed=12)
    ids = (torch.arange(n, device="cuda") % G).to(torch.int32)
    b[0, 7, 3] = math.inf
    b[0, 200:210] = math.nan
    y, m = adapter_oracle(h, w, ids, a, b, s)
    out = fd.adapter_logits(h, w, ids, a, b, s)
    wild = torch.zeros(400, dtype=torch.bool, device="cuda")
    wild[7] = True
    wild[200:210] = True
    touched = (ids == 0)[:, None, None] & wild
    assert not bool(torch.isfinite(out[touched.expand_as(out)]).any())
    clean = ~touched.expand_as(out)
    check_adapter(out[clean], y[clean], m[clean], 64, 16, t)


def test_adapter_logits_beyond_2_31_entries(fd):
    """Offsets of the last tokens pass 32 bits."""
    V, D, n, L = 1100000, 64, 100, 20
    h, w, ids, a, b, s = make_head(n, L, V, D, 8, 2, torch.bfloat16, seed=13)
    out = fd.adapter_logits(h, w, ids, a, b, s)
    assert out.numel() > 2 ** 31
    for i in (0, 98, 99):
        y, m = adapter_oracle(h[i:i + 1], w, ids[i:i + 1], a, b, s)
        check_adapter(out[i:i + 1], y, m, D, 8, torch.bfloat16)


# ------------------------------------------- sequence_logp, preference_loss

def make_candidates(n, L, V, C, seed):
    g = gen(seed)
    pool = torch.randint(0, V, (n, L, 5), generator=g, device="cuda")
    toks = pool.gather(2, torch.randint(0, 5, (n, L, C), generator=g, device="cuda"))
    lens = torch.randint(0, L + 1, (n, C), generator=g, device="cuda", dtype=torch.int32)
    return toks.transpose(1, 2).to(torch.int32).contiguous(), lens


def sequence_oracle(x, toks, lens):
    """Scores and their derivative by the definition, 64 bits, one more token
    (a logit of -inf) standing for every id beyond the vocabulary."""
    n, L, V = x.shape
    lp = torch.log_softmax(x, -1)
    lp = torch.where((x == -math.inf).all(-1, keepdim=True), -math.inf, lp)
    lp = torch.cat([lp, torch.full((n, L, 1), -math.inf, dtype=lp.dtype, device=lp.device)], -1)
    t = toks.long() & 0xFFFFFFFF
    t = torch.where(t >= V, V, t)
    ok = (lens >= 0) & (lens <= L)
    live = (torch.arange(L, device=x.device)[None, None] < lens[..., None]) & ok[..., None]
    each = lp.gather(2, torch.where(live, t, 0).transpose(1, 2)).transpose(1, 2)
    s = torch.where(live, each, 0.0).sum(-1)
    return torch.where(ok, s, math.nan), live, t


def gradient_oracle(x, live, t, w):
    """(gradient, a bound on what its 32-bit terms may be off by)"""
    n, L, V = x.shape
    dead = (x == -math.inf).all(-1, keepdim=True)
    p = torch.where(dead, 0.0, torch.softmax(x, -1))
    part = torch.where(live, w[..., None], 0.0).transpose(1, 2)  # [n, L, C]
    total = part.sum(-1, keepdim=True)
    at = torch.zeros((n, L, V + 1), dtype=x.dtype, device=x.device).scatter_add_(2, t.transpose(1, 2), part)[..., :V]
    mass = torch.zeros((n, L, V + 1), dtype=x.dtype, device=x.device).scatter_add_(2, t.transpose(1, 2),
                                                                                  part.abs())[..., :V]
    at, mass = torch.where(dead, 0.0, at), torch.where(dead, 0.0, mass)
    g = at - total * p
    # W (its 64-bit sum rounded once, and scaled), the row's sum, the
    # exponential and two products; a token's weight; their difference.
    tol = (rel_z(x)[..., None] + (4 * spread(x)[..., None] + 12) * U) * (total * p).abs()
    tol = tol + p * 4 * U * part.abs().sum(-1, keepdim=True) + 4 * U * mass + U * g.abs()
    return g, tol


def check_gradient(dx, x, live, t, w, dtype):
    g, tol = gradient_oracle(x, live, t, w)
    tol = tol + half_step(dtype, g)
    err = (dx.double() - g).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


def score_tol(x, want, live):
    """Each live position: the sum's error; the result is rounded once."""
    per = rel_z(x)[:, None, :] * live
    return per.sum(-1) + U * want.abs() + 2.0 ** -40


SHAPES = [(1, 1, 1, 1), (1, 1, 2, 3), (2, 3, 33, 7), (3, 8, 1001, 10), (1, 24, 4099, 100), (2, 2, 70001, 33),
          (5, 70, 130, 9), (1, 3, 257, 1025), (2, 2, 64, 8192), (60, 4, 515, 40)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,L,V,C", SHAPES)
def test_sequence_logp_and_gradient(fd, t, n, L, V, C):
    x = make_logits(n, L, V, t, seed=V + C, masked=False).requires_grad_()
    toks, lens = make_candidates(n, L, V, C, seed=V)
    lp = fd.sequence_logp(x, toks, lens)
    xd = x.detach().double()
    want, live, at = sequence_oracle(xd, toks, lens)
    assert lp.dtype == torch.float32 and lp.shape == (n, C)
    assert bool(((lp.detach().double() - want).abs() <= score_tol(xd, want, live)).all())
    w = torch.randn((n, C), generator=gen(1), device="cuda")
    (dx,) = torch.autograd.grad(lp, x, w)
    assert dx.dtype == t
    check_gradient(dx, xd, live, at, w.double(), t)


@pytest.mark.parametrize("t", TYPES)
def test_sequence_logp_masked_broken_and_foreign(fd, t):
    """Masked tokens, a row that its mask leaves empty, a row with a NaN, ids
    beyond the vocabulary, lengths out of range, uninitialised tokens behind a
    length."""
    n, L, V, C = 2, 5, 777, 12
    x = make_logits(n, L, V, t, seed=8)
    x[0, 3] = -math.inf
    x[1, 4, 10] = math.nan
    toks, lens = make_candidates(n, L, V, C, seed=8)
    lens[:] = 3
    lens[0, 0], lens[0, 1], lens[0, 2], lens[0, 3] = 0, 6, -1, 4
    lens[1, 0], lens[1, 1], lens[1, 2] = 5, 4, 2147483647
    toks[0, 4, 1] = V
    toks[0, 5, 2] = -1
    toks[0, 6, 3:] = 123456789
    x = x.requires_grad_()
    lp = fd.sequence_logp(x, toks, lens)
    xd = x.detach().double()
    want, live, at = sequence_oracle(xd, toks, lens)
    got = lp.detach().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    fine = torch.isfinite(want)
    assert float(got[0, 0]) == 0.0 and float(got[0, 3]) == -math.inf and math.isnan(float(lp[0, 1].detach()))
    tol = score_tol(xd, torch.where(fine, want, 0.0), live)
    assert bool((torch.where(fine, (got - want).abs(), 0.0) <= tol).all())
    w = torch.randn((n, C), generator=gen(2), device="cuda")
    (dx,) = torch.autograd.grad(lp, x, w)
    # Row (1, 4) has a NaN among its logits and a live candidate: NaN there only.
    assert bool(torch.isnan(dx[1, 4]).any())
    clean = torch.ones((n, L), dtype=torch.bool, device="cuda")
    clean[1, 4] = False
    assert not bool(torch.isnan(dx[clean]).any())
    g, tol = gradient_oracle(torch.where(clean[..., None], xd, 0.0), live, at, w.double())
    err = (dx.double() - g).abs()[clean]
    assert bool((err <= (tol + half_step(t, g))[clean]).all())
    assert not bool(dx[0, 3].any())  # the empty row learns nothing


def preference_oracle(x, toks, lens, ref, c, r, beta, eps, mean):
    n, P = c.shape
    lp, live, at = sequence_oracle(x, toks, lens)
    d = lp - ref.double()
    C = d.shape[1]
    there = (c >= 0) & (r >= 0)
    wrong = there & ((c >= C) | (r >= C))
    ci, ri = c.clamp(0, C - 1).long(), r.clamp(0, C - 1).long()
    z = beta * (d.gather(1, ci) - d.gather(1, ri))
    one = (1 - eps) * torch.nn.functional.softplus(-z, threshold=1e9) + eps * torch.nn.functional.softplus(z, threshold=1e9)
    z, one = torch.where(wrong, math.nan, z), torch.where(wrong, math.nan, one)
    by = 1 / max(1, int(there.sum())) if mean else 1.0
    loss = torch.where(there, one, 0.0).sum() * by
    w = beta * (eps * torch.sigmoid(z) - (1 - eps) * torch.sigmoid(-z)) * by
    w = torch.where(there & ~wrong, w, 0.0)
    g = torch.zeros_like(lp).scatter_add_(1, ci, w).scatter_add_(1, ri, -w)
    return loss, torch.where(there, z, 0.0), g, live, at, by


def make_pairs(n, C, P, seed):
    g = gen(seed)
    c = torch.randint(-1, C, (n, P), generator=g, device="cuda", dtype=torch.int32)
    r = torch.randint(-1, C, (n, P), generator=g, device="cuda", dtype=torch.int32)
    return c, r


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n,L,V,C,P,eps,mean", [(1, 1, 2, 1, 1, 0.0, True), (1, 2, 33, 2, 1, 0.1, False),
                                                (4, 8, 1001, 10, 8, 0.0, True), (2, 24, 4099, 100, 1000, 0.2, True),
                                                (3, 5, 130, 1025, 77, 1.0, False), (2, 3, 515, 40, 0, 0.0, True),
                                                (40, 2, 257, 9, 33, 0.5, True)])
def test_preference_loss_and_gradient(fd, t, n, L, V, C, P, eps, mean):
    beta = 0.3
    x = make_logits(n, L, V, t, seed=C + P, masked=False).requires_grad_()
    toks, lens = make_candidates(n, L, V, C, seed=C)
    xd = x.detach().double()
    lp, live, _ = sequence_oracle(xd, toks, lens)
    ref = (lp + torch.randn((n, C), generator=gen(3), device="cuda")).float()
    c, r = make_pairs(n, C, P, seed=P)
    loss, margin = fd.preference_loss(x, toks, lens, ref, c, r, beta=beta, label_smoothing=eps,
                                      reduction="mean" if mean else "sum")
    assert loss.shape == () and margin.shape == (n, P) and not margin.requires_grad
    want, z, g, live, at, by = preference_oracle(xd, toks, lens, ref, c, r, torch.tensor(beta).float().item(),
                                                 torch.tensor(eps).float().item(), mean)
    tol_lp = (rel_z(xd)[:, None, :] * live).sum(-1).max()  # of any candidate's 64-bit sum
    tol_z = 2 * beta * tol_lp + U * z.abs()
    assert bool(((margin.double() - z).abs() <= tol_z).all())
    pairs = int(((c >= 0) & (r >= 0)).sum())
    # The loss moves by at most |dz| a pair.
    assert abs(float(loss.detach()) - float(want)) <= 2 * beta * float(tol_lp) * pairs * by + 2 * U * abs(float(want))
    (dx,) = torch.autograd.grad(loss * 3.0, x)
    g3 = 3.0 * g
    ref_g, tol = gradient_oracle(xd, live, at, g3)
    # A candidate's weight: each pair's is off by beta/4 of the margin's error
    # and one rounding, and the candidate's sum by one more.
    count = torch.zeros_like(g).scatter_add_(1, c.clamp(0).long(), torch.ones_like(c, dtype=torch.float64)) + \
        torch.zeros_like(g).scatter_add_(1, r.clamp(0).long(), torch.ones_like(r, dtype=torch.float64))
    off = 3.0 * by * count * beta * (beta / 2 * tol_lp + 2 * U) + 2 * U * g3.abs()
    p = torch.softmax(xd, -1)
    part = torch.where(live, off[..., None], 0.0).transpose(1, 2)
    more = torch.zeros((n, L, V + 1), dtype=xd.dtype, device="cuda").scatter_add_(2, at.transpose(1, 2), part)[..., :V]
    tol = tol + more + part.sum(-1, keepdim=True) * p + half_step(t, ref_g)
    err = (dx.double() - ref_g).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


def test_preference_pairs_out_of_range(fd):
    """A slot beyond the candidates makes the loss NaN and moves nothing; a
    negative one is no pair; no pairs at all give 0 and no gradient."""
    x = make_logits(2, 3, 50, torch.float32, seed=1, masked=False).requires_grad_()
    toks, lens = make_candidates(2, 3, 50, 4, seed=1)
    ref = torch.zeros((2, 4), device="cuda")
    c = torch.tensor([[0, -1, 1], [2, 3, -1]], dtype=torch.int32, device="cuda")
    r = torch.tensor([[1, 0, 4], [3, -5, -1]], dtype=torch.int32, device="cuda")
    loss, margin = fd.preference_loss(x, toks, lens, ref, c, r)
    assert math.isnan(float(loss.detach())) and math.isnan(float(margin[0, 2]))
    assert bool(torch.isfinite(margin.flatten()[[0, 1, 3, 4, 5]]).all()) and float(margin[0, 1]) == 0.0
    (dx,) = torch.autograd.grad(loss, x)
    assert bool(torch.isfinite(dx).all())
    none = torch.full_like(c, -1)
    loss, margin = fd.preference_loss(x, toks, lens, ref, none, none)
    assert float(loss.detach()) == 0.0 and not bool(margin.any())
    (dx,) = torch.autograd.grad(loss, x)
    assert not bool(dx.any())


def test_preference_far_margins(fd):
    """Margins of +-1e4 neither overflow nor lose the gradient's limits (0
    and beta)."""
    x = make_logits(1, 2, 20, torch.float32, seed=2, masked=False).requires_grad_()
    toks = torch.tensor([[[1, 2], [3, 4]]], dtype=torch.int32, device="cuda")
    lens = torch.full((1, 2), 2, dtype=torch.int32, device="cuda")
    pair = [torch.tensor([[i]], dtype=torch.int32, device="cuda") for i in (0, 1)]
    for far in (1e5, -1e5):
        ref = torch.tensor([[-far, 0.0]], device="cuda")
        loss, margin = fd.preference_loss(x, toks, lens, ref, *pair, beta=0.1)
        (dx,) = torch.autograd.grad(loss, x)
        if far > 0:
            assert float(loss.detach()) == 0.0 and not bool(dx.any())
        else:
            assert abs(float(loss) + float(margin)) <= 2 * U * abs(float(margin)) and float(dx.abs().max()) > 0.05


@pytest.mark.parametrize("what", ["sequence_logp", "preference_loss"])
def test_gradients_against_differences(fd, what):
    """Directional derivatives by central differences of the operator's own
    values.  f is a sum of log-softmaxes (its third derivative along a unit
    direction is at most 2 per position, L C positions, weights below 4), so
    the difference quotient is off by h^2/6 times that, and by the two values'
    errors over 2h."""
    n, L, V, C, P, h = 2, 4, 60, 6, 5, 2.0 ** -5
    x = make_logits(n, L, V, torch.float32, seed=4, masked=False)
    toks, lens = make_candidates(n, L, V, C, seed=4)
    w = torch.randn((n, C), generator=gen(5), device="cuda").clamp(-3, 3)
    ref = fd.sequence_logp(x, toks, lens) + torch.randn((n, C), generator=gen(6), device="cuda")
    c, r = make_pairs(n, C, P, seed=9)

    def f(v):
        if what == "sequence_logp":
            return (fd.sequence_logp(v, toks, lens).double() * w).sum()
        return fd.preference_loss(v, toks, lens, ref, c, r, beta=0.5, reduction="sum")[0].double()

    xg = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(f(xg), xg)
    xd = x.double()
    lp, live, _ = sequence_oracle(xd, toks, lens)
    value = float((score_tol(xd, lp, live) * 4).sum()) + 4 * U * float(lp.abs().sum())
    for seed in range(4):
        d = torch.randn(x.shape, generator=gen(20 + seed), device="cuda")
        d /= d.norm()
        slope = (f(x + h * d) - f(x - h * d)) / (2 * h)
        # Rounding x + h d moves each logit by at most half a step.
        moved = float(dx.abs().sum()) * U * float(x.abs().max() + 1) / h
        third = 2.0 * n * L * C * 4 * h * h / 6
        assert abs(float(slope) - float((dx.double() * d).sum())) <= third + value / h + moved


def test_gradient_is_the_same_every_time(fd):
    n, L, V, C, P = 3, 20, 5001, 700, 900
    x = make_logits(n, L, V, torch.float32, seed=1, masked=False).requires_grad_()
    toks, lens = make_candidates(n, L, V, C, seed=2)
    ref = torch.randn((n, C), generator=gen(3), device="cuda")
    c, r = make_pairs(n, C, P, seed=4)
    first = None
    for _ in range(4):
        loss, margin = fd.preference_loss(x, toks, lens, ref, c, r)
        (dx,) = torch.autograd.grad(loss, x)
        got = (loss.detach(), margin, dx)
        if first is None:
            first = got
        assert all(torch.equal(p, q) for p, q in zip(first, got))


def test_sequence_logp_beyond_2_31_entries(fd):
    V, L = 2200000, 1000
    x = torch.randn((1, L, V), generator=gen(5), device="cuda", dtype=torch.bfloat16).requires_grad_()
    toks, lens = make_candidates(1, L, V, 6, seed=6)
    lens[:] = torch.tensor([L, L, 3, 0, 990, L], dtype=torch.int32)
    lp = fd.sequence_logp(x, toks, lens)
    w = torch.randn((1, 6), generator=gen(1), device="cuda")
    (dx,) = torch.autograd.grad(lp, x, w)
    for l0 in (0, 980):  # the first and the last positions
        xd = x.detach()[:, l0:l0 + 20].double()
        part = toks[:, :, l0:l0 + 20].contiguous()
        _, live, at = sequence_oracle(xd, part, (lens - l0).clamp(0, 20))
        check_gradient(dx[:, l0:l0 + 20], xd, live, at, w.double(), torch.bfloat16)
    xs = x.detach()[0, :, :].float()
    lse = torch.logsumexp(xs[990:], -1).double()
    del xs
    tail = x.detach()[0, 990:].gather(1, toks[0, 0, 990:, None].long())[:, 0].double() - lse
    short = fd.sequence_logp(x.detach(), toks, torch.full_like(lens, 990))
    # The two scores differ by the last ten positions; each was rounded once.
    tol = 2 * U * float(lp[0, 0].detach().abs()) + 10 * (V / 32 + 200) * U
    assert abs(float(lp[0, 0].detach()) - float(short[0, 0]) - float(tail.sum())) <= tol


def test_sequence_logp_shapes_without_work(fd):
    x = torch.zeros((2, 3, 10), device="cuda", requires_grad=True)
    toks = torch.zeros((2, 0, 3), dtype=torch.int32, device="cuda")
    lp = fd.sequence_logp(x, toks, toks[:, :, 0])
    assert lp.shape == (2, 0)
    (dx,) = torch.autograd.grad(lp.sum(), x)
    assert dx.shape == x.shape and not bool(dx.any())
    empty = torch.zeros((0, 3, 10), device="cuda", requires_grad=True)
    lp = fd.sequence_logp(empty, torch.zeros((0, 4, 3), dtype=torch.int32, device="cuda"),
                          torch.zeros((0, 4), dtype=torch.int32, device="cuda"))
    assert lp.shape == (0, 4)
    z = torch.zeros((0, 4), device="cuda")
    p = torch.zeros((0, 2), dtype=torch.int32, device="cuda")
    loss, margin = fd.preference_loss(empty, torch.zeros((0, 4, 3), dtype=torch.int32, device="cuda"), z.int(), z, p, p)
    assert float(loss.detach()) == 0.0 and margin.shape == (0, 2)


# ------------------------------------------------- streams, graphs, refusals

def _calls(fd, x, h, head, toks, lens, ref, c, r):
    w, ids, a, b, s = head
    leaf = x.detach().requires_grad_()

    def everything():
        y = fd.adapter_logits(h, w, ids, a, b, s, out_dtype=torch.float32)
        top = fd.propose(x, 50)
        lp = fd.sequence_logp(leaf, toks, lens)
        (d1,) = torch.autograd.grad(lp, leaf, ref)
        loss, margin = fd.preference_loss(leaf, toks, lens, ref, c, r)
        (d2,) = torch.autograd.grad(loss, leaf)
        return [y, *top, lp.detach(), d1, loss.detach(), margin, d2]

    return everything


def _inputs(seed, n=3, L=6, V=3001, D=64, r=16, G=4, C=20, P=11):
    x = make_logits(n, L, V, torch.bfloat16, seed, masked=False)
    h, w, ids, a, b, s = make_head(n, L, V, D, r, G, torch.bfloat16, seed)
    toks, lens = make_candidates(n, L, V, C, seed)
    ref = torch.randn((n, C), generator=gen(seed), device="cuda")
    return x, h, (w, ids, a, b, s), toks, lens, ref, *make_pairs(n, C, P, seed)


def test_side_stream(fd):
    args = _inputs(31)
    want = _calls(fd, *args)()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    x, h, head, toks, lens, ref, c, r = args
    w, ids, a, b, s = head
    leaf = x.detach().requires_grad_()
    got = [fd.adapter_logits(h, w, ids, a, b, s, out_dtype=torch.float32, stream=side),
           *fd.propose(x, 50, stream=side)]
    lp = fd.sequence_logp(leaf, toks, lens, stream=side)
    loss, margin = fd.preference_loss(leaf, toks, lens, ref, c, r, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    (d1,) = torch.autograd.grad(lp, leaf, ref)
    (d2,) = torch.autograd.grad(loss, leaf)
    got += [lp.detach(), d1, loss.detach(), margin, d2]
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_captured_and_replayed_on_new_inputs(fd):
    """Two captured graphs, replayed in turn after their inputs have changed,
    while an eager graph of the same leaf lives."""
    first, second = _inputs(41), _inputs(42)
    graphs = []
    for args in (first, second):
        run = _calls(fd, *args)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run()
        graphs.append((g, out, args))
    third = _inputs(43)

    def flat(args):
        return [t for v in args for t in (v if isinstance(v, tuple) else (v,))]

    for g, out, args in graphs:
        for into, new in zip(flat(args), flat(third)):
            into.copy_(new)
    want = _calls(fd, *third)()
    eager_leaf = third[0].detach().requires_grad_()
    alive = fd.sequence_logp(eager_leaf, third[3], third[4])
    for _ in range(2):
        for g, _, _ in graphs:
            g.replay()
    torch.cuda.synchronize()
    for _, out, _ in graphs:
        assert all(torch.equal(p, q) for p, q in zip(want, out))
    del alive


def test_two_threads_at_once(fd):
    """Calls from two threads on streams of their own give what one thread
    gets, whatever sizes the other one asks for."""
    import threading
    sets = [_inputs(71), _inputs(72, n=5, L=3, V=1201, D=128, r=8, G=2, C=300, P=40)]
    want = [_calls(fd, *a)() for a in sets]
    torch.cuda.synchronize()
    wrong = []

    def work(which):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            run = _calls(fd, *sets[which])
            for _ in range(20):
                got = run()
                stream.synchronize()
                if not all(torch.equal(p, q) for p, q in zip(want[which], got)):
                    wrong.append(which)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_a_weight_that_is_no_number_stays_in_its_rows(fd):
    """An upstream gradient of NaN makes NaN of the positions that its
    candidate reaches, and of nothing else."""
    x = make_logits(2, 6, 333, torch.float32, seed=3, masked=False).requires_grad_()
    toks, lens = make_candidates(2, 6, 333, 9, seed=3)
    lens[0, 4], lens[1, 4] = 3, 0
    lp = fd.sequence_logp(x, toks, lens)
    w = torch.randn((2, 9), generator=gen(3), device="cuda")
    (clean,) = torch.autograd.grad(lp, x, w, retain_graph=True)
    w[0, 4] = math.nan
    (dx,) = torch.autograd.grad(lp, x, w)
    assert bool(torch.isnan(dx[0, :3]).all())
    assert torch.equal(dx[0, 3:], clean[0, 3:]) and torch.equal(dx[1], clean[1])


def test_hidden_search_of_no_requests(fd, tmp_path):
    import flashtrie
    t = flashtrie.Trie()
    t.build(token_rows=[[1, 2], [3]])
    t.init_tbs_gpu(1, max_num_topk=8, max_num_outpos=4, max_num_out_beams=4)
    h, w, ids, a, b, s = make_head(1, 4, 50, 64, 8, 2, torch.bfloat16, seed=1)
    beams = torch.full((0, 4), 4, dtype=torch.int32, device="cuda")
    out = fd.bs_tbs_hidden(t, beams, h[:0], w, 8, -10.0, -40.0, 1.0, False, ids[:0], a, b, s)
    assert out[0].shape == (0,)
    with pytest.raises(ValueError):
        fd.bs_tbs_hidden(t, beams, h, w, 8, -10.0, -40.0, 1.0, False)


def test_python_refusals(fd):
    x, h, (w, ids, a, b, s), toks, lens, ref, c, r = _inputs(51)
    bad_adapter = [
        (h.float(), w, ids, a, b, s), (h, w.to(torch.float16), ids, a, b, s), (h, w[:, :32].contiguous(), ids, a, b, s),
        (h, w, ids.long(), a, b, s), (h, w, ids[:2], a, b, s), (h, w, ids, a[:, :, :32].contiguous(), b, s),
        (h, w, ids, a, b[:, 1:].contiguous(), s), (h, w, ids, a, b, s[:1]), (h, w, ids, a[:0], b[:0], s[:0]),
        (h, w, ids, None, None, None), (h, w, None, a, b, None), (h, w, None, None, None, s),
        (h.transpose(0, 1), w, ids, a, b, s), (h[:, :0], w, ids, a, b, s), (h, w.t().contiguous().t(), ids, a, b, s)]
    for args in bad_adapter:
        with pytest.raises(ValueError):
            fd.adapter_logits(*args)
    with pytest.raises(ValueError):
        fd.adapter_logits(h, w, ids, a, b, s, out_dtype=torch.float16)
    with pytest.raises(ValueError):
        fd.adapter_logits(h, w.detach().requires_grad_(), ids, a, b, s)
    with pytest.raises(RuntimeError):  # D is no multiple of 8
        fd.adapter_logits(h[:, :, :60].contiguous(), w[:, :60].contiguous())
    with torch.no_grad():
        fd.adapter_logits(h, w.detach().requires_grad_(), ids, a, b, s)
    for k, order in ((0, "id"), (8193, "id"), (5, "best")):
        with pytest.raises(ValueError):
            fd.propose(x, k, order=order)
    for bad in (x.double(), x[0], x.transpose(1, 2), x[:, :, :0]):
        with pytest.raises(ValueError):
            fd.propose(bad, 3)
    with pytest.raises(ValueError):
        fd.propose(x.detach().requires_grad_(), 3)
    for args in [(x.double(), toks, lens), (x, toks.long(), lens), (x, toks, lens.long()), (x, toks[:, :, :2], lens),
                 (x, toks[:, 1:].contiguous(), lens), (x, toks[:2], lens[:2]), (x[:, :, ::2], toks, lens)]:
        with pytest.raises(ValueError):
            fd.sequence_logp(*args)
        with pytest.raises(ValueError):
            fd.preference_loss(*args, ref, c, r)
    for args in [(ref.double(), c, r), (ref[:, 1:].contiguous(), c, r), (ref, c.long(), r), (ref, c[:, :2].contiguous(), r),
                 (ref.detach().requires_grad_(), c, r)]:
        with pytest.raises(ValueError):
            fd.preference_loss(x, toks, lens, *args)
    for kw in (dict(beta=math.inf), dict(beta=1e300), dict(label_smoothing=1.5), dict(reduction="none")):
        with pytest.raises(ValueError):
            fd.preference_loss(x, toks, lens, ref, c, r, **kw)


def test_gradients_accumulate_with_other_terms(fd):
    """The loss in place among other terms of an objective: the leaf's
    gradient is the sum, for the search's own layout of results."""
    x, _, _, toks, lens, ref, c, r = _inputs(61)
    leaf = x.float().requires_grad_()
    (fd.preference_loss(leaf, toks, lens, ref, c, r)[0] * 2 + (fd.sequence_logp(leaf, toks, lens) * ref).sum()).backward()
    a = x.float().requires_grad_()
    (d1,) = torch.autograd.grad(fd.preference_loss(a, toks, lens, ref, c, r)[0] * 2, a)
    (d2,) = torch.autograd.grad(fd.sequence_logp(a, toks, lens), a, ref)
    assert torch.equal(leaf.grad, d1 + d2)
    loss, _ = fd.preference_loss(a, toks, lens, ref, c, r)
    loss /= 4
    loss.backward()
    assert torch.equal(a.grad, torch.autograd.grad(fd.preference_loss(a, toks, lens, ref, c, r)[0] / 4, a)[0])


# ------------------------------------------------------------ the whole path

def test_from_hidden_states_to_a_preference_step(fd, tmp_path):
    """Hidden states -> logits with adapters -> proposals -> search -> scores
    of the results -> preference loss and gradient, against the oracle search
    on the same proposals and 64-bit scores."""
    import flashtrie
    import workload as W
    from oracle.oracle import OracleTrie
    cfg = dict(W.CONFIGS[1])
    n, L, V, K, D = 6, cfg["L"], cfg["vocab"], cfg["K"], 256
    tok, off = W.gen_keys(30000, V, cfg["len_lo"], cfg["len_hi"], cfg["zipf"], seed=77)
    t = flashtrie.Trie()
    t.build_flat(tok, off)
    path = str(tmp_path / "p.bin")
    t.save(path)
    t.init_tbs_gpu(n, max_num_topk=K, max_num_outpos=L, max_num_out_beams=cfg["beam"])
    h, w, ids, a, b, s = make_head(n, L, V, D, 8, 3, torch.bfloat16, seed=78)
    # Each request's hidden states point to the tokens of two keys, far enough
    # that they are among the K best of their positions.
    for i in range(n):
        for key in (tok[off[j]:off[j + 1]] for j in (100 * i, 100 * i + 50)):
            for l, v in enumerate(key[:L]):
                h[i, l] = h[i, l] + 16 * w[int(v)]
    beams = torch.full((n, L), cfg["beam"], dtype=torch.int32, device="cuda")
    out = fd.bs_tbs_hidden(t, beams, h, w, K, -30.0, -200.0, 0.0, False, ids, a, b, s)
    logits = fd.adapter_logits(h, w, ids, a, b, s, out_dtype=torch.float32)
    y, m = adapter_oracle(h, w, ids, a, b, s)
    check_adapter(logits, y, m, D, 8, torch.bfloat16)
    top = fd.propose(logits, K)
    check_propose(fd, logits, K, "id")
    sents, lpns = fd.to_lists(out)
    o = OracleTrie(path)
    for i in range(n):
        ids_i = top[0][i].cpu().numpy().view(np.uint32)
        want = o.tbs([cfg["beam"]] * L, ids_i, top[1][i].cpu().numpy(), -30.0, -200.0, 0.0, False)
        assert sents[i] == want[0] and lpns[i] == want[1]
    count, lpn, lens, toks = out
    assert int(count.min()) >= 2
    leaf = logits.detach().requires_grad_()
    lp = fd.sequence_logp(leaf, toks, lens)
    want, live, at = sequence_oracle(logits.double(), toks, lens)
    assert bool(((lp.detach().double() - want).abs() <= score_tol(logits.double(), want, live)).all())
    # Without a length norm a result's score is its log-probability.
    filled = torch.arange(lpn.shape[1], device="cuda")[None] < count[:, None]
    near = score_tol(logits.double(), want, live) + L * (rel_z(logits.double()).max() + 64 * U)
    assert bool((torch.where(filled, (lpn - want).abs(), 0.0) <= near).all())
    ref = lp.detach() * 0.9
    best = (count - 1)[:, None].to(torch.int32)
    worst = torch.zeros_like(best)
    loss, margin = fd.preference_loss(leaf, toks, lens, ref, best, worst)
    (dx,) = torch.autograd.grad(loss, leaf)
    with torch.no_grad():
        after, more = fd.preference_loss(leaf - 20.0 * dx, toks, lens, ref, best, worst)
    assert bool((more > margin).all())  # a step down the gradient prefers the chosen ones more

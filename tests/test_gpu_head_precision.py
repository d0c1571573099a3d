"""How exact the model-side operators are, each property with data that leaves
no room for anything else: sums whose terms are all 1, weights of very
different sizes, low-rank values far from 1.

Tolerances, derived here (U = 2^-24, half a step of f32):
  - logits of 0 and -inf alone have exponentials of exactly 1 and 0, so that a
    softmax sum is a count, exact in f32 up to 2^24 in any order; a 64-bit
    logarithm is off by a step at most;
  - a weight of a preference pair is computed in 64 bits, rounded once as the
    candidate's gradient, once with the factors and once in the row: 3 U, and
    one more for the mean's factor; an upstream weight of a score is rounded
    twice, and the sums lose 2^-48 of their largest weight at most;
  - low-rank values: 2 (D + 2) U of their products' absolute sum, then what the
    16-bit parts lose (LOSS), then 2 (parts r + 2) U of sum |u b| for the second
    product.
"""
import math

import pytest
import torch

from test_gpu_head_ops import HALVES, TYPES, U, gen, half_step, make_head, make_logits, spread

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fd(built):
    import flashtrie_device
    return flashtrie_device


# ------------------------------------------------------- weights of all sizes

def spiked(C):
    """Logits [1, 1, C + 1] of which the first takes all of the probability
    (the others have e^-60 of it), and a candidate for each of the others: its
    log-probability is -60 (off by 1e-23), its token no other's."""
    x = torch.zeros((1, 1, C + 1), device="cuda")
    x[..., 0] = 60.0
    toks = torch.arange(1, C + 1, device="cuda", dtype=torch.int32).view(1, C, 1)
    return x, toks, torch.ones((1, C), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("lo,hi,P,absent", [(25, 40, 1000, 0), (36, 50, 200, 0), (36, 60, 200, 0),
                                            (-5, 75, 1000, 0), (0, 40, 1, 0), (-5, 60, 3001, 0), (10, 60, 8191, 1),
                                            (20, 30, 3, 200000)])
@pytest.mark.parametrize("reduction", ["sum", "mean"])
def test_pair_weights_of_any_margin(fd, lo, hi, P, absent, reduction):
    """Each pair's candidate gets the pair's own weight, however far apart the
    pair is, whatever other pairs there are."""
    beta = torch.tensor(0.1).item()
    x, toks, lens = spiked(P + 1)
    lens[0, P] = 0  # the other side of all pairs
    z = torch.linspace(lo, hi, P, dtype=torch.float64, device="cuda")
    ref = torch.zeros((1, P + 1), device="cuda")
    ref[0, :P] = (-60.0 - z / beta).float()
    z = beta * (-60.0 - ref[0, :P].double())
    c = torch.full((1, P + absent), -1, dtype=torch.int32, device="cuda")
    r = torch.full_like(c, P)
    at = torch.arange(P, device="cuda") * (1 + absent // P)
    c[0, at] = torch.arange(P, device="cuda", dtype=torch.int32)
    leaf = x.requires_grad_()
    loss, margin = fd.preference_loss(leaf, toks, lens, ref, c, r, beta=beta, reduction=reduction)
    assert bool(((margin[0, at].double() - z).abs() <= U * z.abs()).all())
    (dx,) = torch.autograd.grad(loss, leaf)
    want = -beta * torch.sigmoid(-z) / (P if reduction == "mean" else 1)
    # The softmax part of each entry: the row's whole weight times e^-60.
    tol = 4 * U * want.abs() + want.abs().sum() * 2 * math.exp(-60) + 2.0 ** -126
    err = (dx[0, 0, 1:P + 1].double() - want).abs()
    assert bool((err <= tol).all()), float((err / want.abs()).max())


@pytest.mark.parametrize("share", [1, 2, 50])
def test_token_weights_of_any_size(fd, share):
    """Weights 14 powers of ten apart in one row, `share` candidates of one
    size with each token: every token's sum is as exact as its own weights."""
    C = 1000
    x, toks, lens = spiked(C)
    toks = ((toks - 1) // share + 1).contiguous()
    size = 10.0 ** (-14 * torch.rand((C // share, 1), generator=gen(1), device="cuda", dtype=torch.float64))
    w = (size * (0.5 + torch.rand((C // share, share), generator=gen(2), device="cuda", dtype=torch.float64))).float()
    w *= torch.where(torch.rand(w.shape, generator=gen(3), device="cuda") < 0.5, -1.0, 1.0)
    leaf = x.requires_grad_()
    (dx,) = torch.autograd.grad(fd.sequence_logp(leaf, toks, lens), leaf, w.view(1, C))
    want = w.double().sum(1)
    tol = 3 * U * want.abs() + 2.0 ** -48 * w.double().abs().sum(1) + w.double().abs().sum() * 2 * math.exp(-60)
    err = (dx[0, 0, 1:C // share + 1].double() - want).abs()
    assert bool((err <= tol).all()), float((err / w.double().abs().sum(1)).max())


# ------------------------------------------------------------ low-rank values

# What the 16-bit parts of a low-rank value lose, relative, by (type, f32 out).
LOSS = {(torch.bfloat16, False): 2.0 ** -17, (torch.bfloat16, True): 2.0 ** -26,
        (torch.float16, False): 2.0 ** -23, (torch.float16, True): 2.0 ** -23}
# n, L, G: one request; requests of a few adapters; an adapter for every token.
FORMS = [(1, 5, 1), (6, 20, 3), (40, 1, 40)]


@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("n,L,G", FORMS)
@pytest.mark.parametrize("scale", [1e-30, 1e-6, 2.0 ** -9, 1.0, 1e5, 1e30])
@pytest.mark.parametrize("shared", [False, True])
def test_low_rank_values_of_any_size(fd, t, n, L, G, scale, shared):
    """The low-rank part beside a shared projection or alone: as exact where
    its values are tiny or beyond the type's largest as where they are near 1,
    and the same in every form that a batch may take."""
    D, V, r = 64, 300, 8
    h, w, ids, a, b, s = make_head(n, L, V, D, r, G, t, seed=7)
    ids = (torch.arange(n, device="cuda") % G).to(torch.int32)
    if not shared:
        w = torch.zeros_like(w)
    check_low_rank(fd, h, w, ids, a, b, s * scale)


def check_low_rank(fd, h, w, ids, a, b, s):
    t, D, r = h.dtype, h.shape[2], a.shape[1]
    at = ids.long().clamp(min=0)
    hd, ad, bd = h.double(), a.double()[at], b.double()[at]
    f = torch.where(ids >= 0, s.double()[at], 0.0)[:, None, None]
    u = (hd @ ad.transpose(1, 2)) * f
    y = hd @ w.double().T + u @ bd.transpose(1, 2)
    shared_mass = hd.abs() @ w.double().abs().T
    u_mass = (hd.abs() @ ad.abs().transpose(1, 2)) * f @ bd.abs().transpose(1, 2)
    mass = u.abs() @ bd.abs().transpose(1, 2)
    for out_t in (t, torch.float32):
        out = fd.adapter_logits(h, w, ids, a, b, s, out_dtype=out_t).double()
        parts = LOSS[t, out_t == torch.float32]
        tol = 2 * (D + 3 * r + 2) * U * (shared_mass + mass) + 2 * (D + 2) * U * u_mass + parts * mass
        if t == torch.float16:
            # Two f16 parts leave up to 2^-25 behind, absolute; tokens whose
            # largest value is below 2^-8 take no part in that.
            near = (u.abs().amax(-1) >= 2.0 ** -8)[..., None]
            tol = tol + near * 2.0 ** -25 * bd.abs().sum(-1)[:, None]
        tol = tol + half_step(out_t, y)
        beyond = y.abs() + tol > torch.finfo(out_t).max
        assert bool((torch.isfinite(out) | beyond).all())
        err = torch.where(beyond, 0.0, (out - y).abs())
        assert bool((err <= tol).all()), float((err / (mass + shared_mass)).max())


@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("n,L,V,D,r,G", [(1, 300, 8001, 72, 64, 1), (1, 7, 80000, 64, 16, 2), (20, 20, 76000, 136, 40, 6),
                                         (2, 30, 76032, 1160, 72, 3), (9, 33, 777, 64, 256, 2), (64, 4, 515, 64, 32, 9)])
def test_tokens_of_all_sizes_side_by_side(fd, t, n, L, V, D, r, G):
    """Tokens whose low-rank values the 16-bit parts hold beside tokens whose
    values they do not, in several tiles and slices, requests without an
    adapter among them."""
    h, w, ids, a, b, s = make_head(n, L, V, D, r, G, t, seed=11)
    size = 2.0 ** (torch.randint(0, 3, (n, L, 1), generator=gen(12), device="cuda") * 12 - 12).double()
    h = (h.double() * size).to(t)
    b = (b.double() * 2.0 ** -6).to(t)
    if n == 1:
        ids = torch.zeros_like(ids)
    check_low_rank(fd, h, w, ids, a, b, s * 2.0 ** 5)


@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("n,L,G", FORMS)
def test_low_rank_parts_hold_what_they_say(fd, t, n, L, G):
    """One product alone: h, A and B are single ones, so that the logit is the
    adapter's scale, all of its 24 bits but what the parts lose."""
    D, V, r = 64, 130, 16
    h = torch.zeros((n, L, D), dtype=t, device="cuda")
    h[..., 3] = 1.0
    a = torch.zeros((G, r, D), dtype=t, device="cuda")
    a[:, 5, 3] = 1.0
    b = torch.zeros((G, V, r), dtype=t, device="cuda")
    b[:, :, 5] = 1.0
    s = torch.rand(G, generator=gen(4), device="cuda") + 0.5
    ids = (torch.arange(n, device="cuda") % G).to(torch.int32)
    out = fd.adapter_logits(h, torch.zeros((V, D), dtype=t, device="cuda"), ids, a, b, s, out_dtype=torch.float32)
    want = s.double()[ids.long()][:, None, None]
    assert bool(((out.double() - want).abs() <= LOSS[t, True] * want).all())


def test_long_sums_are_two_of_half_the_length(fd):
    """f32 logits, all products positive: a sum of 2048 is off by no more than
    one of 1024 (as many partial sums are cut in each of its halves; a quarter
    is left for the spread of the mean)."""
    off = []
    for D in (1024, 2048):
        h = torch.randn((1, 16, D), generator=gen(5), device="cuda").abs().to(torch.bfloat16)
        w = torch.randn((4096, D), generator=gen(6), device="cuda").abs().to(torch.bfloat16)
        y = h.double() @ w.double().T
        off.append(abs(float(((fd.adapter_logits(h, w, out_dtype=torch.float32).double() - y) / y).mean())))
    assert off[1] <= 1.25 * off[0], off


# ------------------------------------------------------------------- counts

def counted(V, L, t, seed):
    """Logits of 0 and -inf, the number of zeros of each row, and where one is."""
    x = torch.zeros((1, L, V), device="cuda")
    x[torch.rand((1, L, V), generator=gen(seed), device="cuda") < 0.3] = -math.inf
    x[0, 0] = 0.0
    live = torch.randint(0, V, (L,), generator=gen(seed + 1), device="cuda")
    x[0, torch.arange(L), live] = 0.0
    return x.to(t), (x == 0).sum(-1)[0].double(), live


SIZES = [(1, 3), (5, 2), (777, 24), (4099, 24), (100003, 24), (100003, 2), (400009, 3), (2200000, 2)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("V,L", SIZES)
def test_log_sums_count_every_value_once(fd, t, V, L):
    """A value left out or taken twice anywhere in a row changes the count. The
    margin shows the 64-bit score less its own rounding to f32."""
    x, count, live = counted(V, L, t, seed=V)
    want = -float(count.log().sum())
    toks = live.to(torch.int32).view(1, 1, L).expand(1, 2, L).contiguous()
    lens = torch.tensor([[L, 0]], dtype=torch.int32, device="cuda")
    ref = torch.tensor([[want, 0.0]], device="cuda")
    pair = [torch.tensor([[i]], dtype=torch.int32, device="cuda") for i in (0, 1)]
    leaf = x.requires_grad_()
    _, margin = fd.preference_loss(leaf, toks, lens, ref, *pair, beta=1.0)
    rest = want - float(ref[0, 0].double())
    assert abs(float(margin) - rest) <= L * 16 * 2.0 ** -52 + U * abs(rest)
    lp = fd.sequence_logp(leaf, toks, lens)
    assert abs(float(lp[0, 0].detach()) - want) <= U * abs(want) + L * 16 * 2.0 ** -52
    # Every zero's gradient is -1 / count (the token's, 1 more): the division
    # and the product are rounded, then the result.
    (dx,) = torch.autograd.grad(lp[0, 0], leaf)
    g = torch.where(x.detach() == 0, (-1 / count)[None, :, None], 0.0)
    g[0, torch.arange(L), live] += 1.0
    tol = 3 * U * g.abs() + half_step(t, g)
    assert bool(((dx.double() - g).abs() <= tol).all())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("V,L", SIZES[:-1])
def test_proposals_count_every_value_once(fd, t, V, L):
    x, count, _ = counted(V, L, t, seed=V + 3)
    _, lps = fd.propose(x, 1)
    want = -count.log()
    tol = 2 * U * want.abs()  # one step of the logarithm
    assert V == 1 or bool((tol < 1 / count).all())
    assert bool(((lps[0, :, 0].double() - want).abs() <= tol).all())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("V,R,seed", [(1001, 400, 1), (32000, 100, 2), (500009, 60, 3), (2200000, 24, 4)])
def test_log_sums_do_not_lean(fd, t, V, R, seed):
    """The mean error over many rows. The base-2 exponential is 5e-8 low on
    average over its argument's fractions, and nothing that the joins do adds
    to that; 3 / sqrt(R) of a sum's own spread (its terms' errors and a few dozen
    roundings, 2 U) is left for the mean."""
    x = torch.randn((R, 1, V), generator=gen(seed), device="cuda") * 2
    x = (x - 0.3 * torch.log1p(torch.arange(V, device="cuda", dtype=torch.float32))).to(t)
    top = x[:, 0].argmax(-1)
    pair = [torch.full((R, 1), i, dtype=torch.int32, device="cuda") for i in (0, 1)]
    toks = top.to(torch.int32).view(R, 1, 1).expand(R, 2, 1).contiguous()
    lens = torch.tensor([1, 0], dtype=torch.int32, device="cuda").expand(R, 2).contiguous()
    want = torch.stack([torch.log_softmax(x[i, 0].double(), -1)[top[i]] for i in range(R)])
    ref = torch.stack([want.float(), torch.zeros(R, device="cuda")], 1).contiguous()
    _, margin = fd.preference_loss(x, toks, lens, ref, *pair, beta=1.0)
    off = margin[:, 0].double() - (want - ref[:, 0].double())
    assert abs(float(off.mean())) <= 5e-8 + 3 / math.sqrt(R) * 2 * U, (float(off.mean()), float(off.std()))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("V,L", [(4099, 24), (100003, 24), (100003, 2), (300001, 3)])
def test_log_sums_of_ordinary_rows(fd, t, V, L):
    """A thread of 512 adds V / 512 values and a few more for the row's ends and
    the joins; an exponential's argument is off by 2 U of the spread, the
    exponential by 4 U."""
    x = make_logits(1, L, V, t, seed=V + L, masked=False)
    xd = x.double()
    lp = torch.log_softmax(xd, -1)
    top = xd.argmax(-1)
    want = lp.gather(2, top[..., None])[0, :, 0]
    tol = (4 * spread(xd)[0] + 8 + V / 512 + 112) * U + 2 * U * want.abs()
    _, got = fd.propose(x, 1)
    assert bool(((got[0, :, 0].double() - want).abs() <= tol).all())
    toks = top.view(L, 1, 1).to(torch.int32)
    score = fd.sequence_logp(x.view(L, 1, V), toks, torch.ones((L, 1), dtype=torch.int32, device="cuda"))
    assert bool(((score[:, 0].double() - want).abs() <= tol).all())

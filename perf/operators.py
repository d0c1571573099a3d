"""Measured cases of the device operators around the trie-constrained search.

The search takes per-position top-k proposals and answers with scored
sequences.  The operators measured here are the model-side steps next to it:
  logits    the vocabulary projection of many requests at once, each request
            with a low-rank adapter of its own beside the shared weight;
  propose   log-softmax over the vocabulary and its top k: the search's
            topk_id and topk_logp;
  score     log-probabilities of candidate sequences (the search's results)
            under the model's logits, forward alone or with the gradient;
  prefer    the preference loss on pairs of candidates (paired log ratios
            against a reference), with the gradient of the logits.

`run` makes one pass: in elementary torch operations when `own` is false, by
the calls of `flashtrie_device` when it is true.
"""
import math
import os
import sys

import torch

own = False

FLT_MAX = 3.4028234663852886e38
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _device_api():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-trie_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import flashtrie_device
    return flashtrie_device


# ---------------------------------------------------------------- cases

def _logits(n, L, V, D, r, G, dtype, out):
    return dict(op="logits", n=n, L=L, V=V, D=D, r=r, G=G, dtype=dtype, out=out)


def _propose(n, L, V, k, dtype, order):
    return dict(op="propose", n=n, L=L, V=V, k=k, dtype=dtype, order=order)


def _score(n, L, V, C, dtype, grad):
    return dict(op="score", n=n, L=L, V=V, C=C, dtype=dtype, grad=grad)


def _prefer(n, L, V, C, P, dtype, smoothing):
    return dict(op="prefer", n=n, L=L, V=V, C=C, P=P, dtype=dtype, smoothing=smoothing)


def listed():
    return [
        # One request of the small configuration (vocabulary 32,000, 8 positions): latency.
        dict(name="logits_one_32k", **_logits(1, 8, 32000, 512, 8, 4, "bf16", "bf16")),
        # Single tokens of 37 requests, most of them with an adapter that no other has.
        dict(name="logits_tokens_32k", **_logits(37, 1, 32000, 1024, 16, 40, "fp16", "fp16")),
        # The mid-size vocabulary for a handful of requests, logits kept in 32 bits for the log-softmax.
        dict(name="logits_500k_fp32", **_logits(8, 16, 500000, 768, 16, 8, "bf16", "fp32")),
        # One request of the large vocabulary (20 positions): the weight's bytes are the time.
        dict(name="logits_one_2m", **_logits(1, 20, 2200000, 1024, 16, 8, "bf16", "bf16")),
        # A full batch of 64 requests with 16 adapters: the matrix products are the time.
        dict(name="logits_batch_500k", **_logits(64, 20, 500000, 2048, 64, 16, "bf16", "bf16")),
        # Proposals of one request of the small configuration: latency.
        dict(name="propose_one_32k", **_propose(1, 8, 32000, 64, "fp32", "id")),
        # Proposals of one request of the large configuration (K = 1000).
        dict(name="propose_one_2m", **_propose(1, 20, 2200000, 1000, "bf16", "id")),
        # Proposals of a batch of the mid-size configuration, an odd vocabulary, best first.
        dict(name="propose_batch_500k", **_propose(16, 16, 500009, 256, "fp32", "logp")),
        # A reference model's scores of 100 results for each of 4 requests, an odd vocabulary.
        dict(name="score_500k", **_score(4, 16, 500009, 100, "fp32", False)),
        # Scores with the gradient, small vocabulary: a training step's latency.
        dict(name="score_grad_32k", **_score(2, 8, 32000, 10, "fp16", True)),
        # Preference pairs among the results of the small configuration, a batch of 16.
        dict(name="prefer_32k", **_prefer(16, 8, 32000, 10, 8, "fp32", 0.1)),
        # Pairs among 1000 results of two requests of the large configuration (24 positions).
        dict(name="prefer_2m", **_prefer(2, 24, 2200000, 1000, 1000, "bf16", 0.0)),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logits", "propose", "score", "prefer"])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    L = rng.randint(1, 24)
    if op == "logits":
        dtype = rng.choice(["bf16", "fp16"])
        V, D = _spread(rng, 1000, 2200000), 8 * _spread(rng, 8, 256)
        while V * D > 2000000000:
            V, D = _spread(rng, 1000, 2200000), 8 * _spread(rng, 8, 256)
        n = _spread(rng, 1, max(1, min(256, 300000000 // (V * L))))
        r = 8 * rng.randint(1, 8)
        G = _spread(rng, 1, max(1, min(64, 300000000 // (V * r))))
        return _logits(n, L, V, D, r, G, dtype, rng.choice([dtype, "fp32"]))
    V = _spread(rng, 500, 2200000)
    n = _spread(rng, 1, max(1, min(64, 100000000 // (V * L))))
    if op == "propose":
        return _propose(n, L, V, _spread(rng, 1, min(V, 2000)), dtype, rng.choice(["id", "logp"]))
    C = _spread(rng, 1, 1000)
    if op == "score":
        return _score(n, L, V, C, dtype, rng.random() < 0.5)
    return _prefer(n, L, V, max(2, C), _spread(rng, 1, 1000), dtype, rng.choice([0.0, 0.1]))


# ---------------------------------------------------------------- inputs

def _model_logits(c, g):
    """Logits N(0, 2) falling with the token id, as vocabularies ordered by
    frequency have them; every 97th token of the vocabulary masked away."""
    n, L, V = c["n"], c["L"], c["V"]
    x = torch.randn((n, L, V), generator=g, device="cuda") * 2
    x -= 0.3 * torch.log1p(torch.arange(V, device="cuda", dtype=torch.float32))
    if c["op"] == "propose":
        x[..., torch.arange(V, device="cuda") % 97 == 96] = float("-inf")
    return x.to(DTYPES[c["dtype"]])


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n, L, V = c["n"], c["L"], c["V"]
    if c["op"] == "logits":
        t, D, r, G = DTYPES[c["dtype"]], c["D"], c["r"], c["G"]
        s = dict(c=c)
        s["hidden"] = torch.randn((n, L, D), generator=g, device="cuda").to(t)
        s["weight"] = (torch.randn((V, D), generator=g, device="cuda", dtype=torch.float32) / math.sqrt(D)).to(t)
        s["lora_a"] = (torch.randn((G, r, D), generator=g, device="cuda") / math.sqrt(D)).to(t)
        s["lora_b"] = (torch.randn((G, V, r), generator=g, device="cuda") * 0.3).to(t)
        s["scales"] = torch.rand(G, generator=g, device="cuda") + 0.5
        # One request in eight has no adapter.
        ids = torch.randint(0, G, (n,), generator=g, device="cuda", dtype=torch.int32)
        s["adapter_ids"] = torch.where(torch.rand(n, generator=g, device="cuda") < 0.125, -1, ids).to(torch.int32)
        return s
    s = dict(c=c, logits=_model_logits(c, g))
    if c["op"] == "propose":
        return s
    C = c["C"]
    # Beams share tokens: a candidate's token at each position is one of a
    # few dozen, the first ones far more often; one slot in ten is empty.
    pool = (torch.rand((n, L, 64), generator=g, device="cuda") ** 3 * V).long().clamp_(max=V - 1)
    pick = (torch.rand((n, L, C), generator=g, device="cuda") ** 3 * 64).long().clamp_(max=63)
    s["tokens"] = pool.gather(2, pick).transpose(1, 2).to(torch.int32).contiguous()
    lens = torch.randint(1, L + 1, (n, C), generator=g, device="cuda")
    s["lengths"] = torch.where(torch.rand((n, C), generator=g, device="cuda") < 0.1, 0, lens).to(torch.int32)
    if c["op"] == "score":
        s["g"] = torch.randn((n, C), generator=g, device="cuda")
        return s
    P = c["P"]
    lp = _plain_score(s["logits"], s["tokens"], s["lengths"])[0]
    s["ref"] = (lp + torch.randn((n, C), generator=g, device="cuda")).float()
    a = torch.randint(0, C, (n, P), generator=g, device="cuda")
    b = (a + torch.randint(1, C, (n, P), generator=g, device="cuda")) % C
    s["chosen"] = torch.where(torch.rand((n, P), generator=g, device="cuda") < 0.1, -1, a).to(torch.int32)
    s["rejected"] = b.to(torch.int32)
    return s


BETA = 0.1


# ---------------------------------------------------------------- plain forms

def _plain_logits(s):
    c = s["c"]
    n, L, D, r, G = c["n"], c["L"], c["D"], c["r"], c["G"]
    x = s["hidden"].float().view(n * L, D)
    y = x @ s["weight"].float().T
    # The low-rank parts as one product: each token's r values in its
    # adapter's columns, zeros in those of the others.
    u = (x @ s["lora_a"].float().view(G * r, D).T).view(n, L, G, r)
    own_cols = (s["adapter_ids"][:, None] == torch.arange(G, device="cuda")[None, :]).float() * s["scales"]
    u = (u * own_cols[:, None, :, None]).view(n * L, G * r)
    y += u @ s["lora_b"].float().transpose(1, 2).reshape(G * r, c["V"])
    return y.to(DTYPES[c["out"]]).view(n, L, c["V"])


def _plain_propose(s):
    c = s["c"]
    x = s["logits"].float()
    m = x.amax(-1, keepdim=True)
    logz = (x - m).exp().sum(-1, keepdim=True).log()
    val, idx = torch.sort(x, dim=-1, descending=True, stable=True)
    val, idx = val[..., :c["k"]], idx[..., :c["k"]]
    lp = (val - m) - logz
    none = val == float("-inf")
    idx = torch.where(none, -1, idx)
    lp = torch.where(none, -FLT_MAX, lp)
    if c["order"] == "id":
        at = torch.argsort(torch.where(none, c["V"], idx), dim=-1, stable=True)
        idx, lp = idx.gather(-1, at), lp.gather(-1, at)
    return idx.to(torch.int32), lp


def _plain_score(logits, tokens, lengths):
    """(scores in 64 bits, probabilities, tokens by position, positions in
    use): a preference's margin is a small difference of long sums."""
    x = logits.float()
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    z = e.sum(-1, keepdim=True)
    L = x.shape[1]
    live = torch.arange(L, device=x.device)[None, :, None] < lengths[:, None, :]
    tok = torch.where(live, tokens.transpose(1, 2), 0).long()
    lp = x.gather(2, tok).double() - m.double() - z.double().log()
    lp = torch.where(live, lp, 0.0).sum(1)
    return lp, e.div_(z), tok, live


def _plain_gradient(p, tok, live, g):
    """Gradient of sum(g * scores): each candidate's share at its tokens, less
    the position's whole share spread by the probabilities."""
    part = torch.where(live, g[:, None, :], 0.0)
    d = p.mul_(-part.sum(-1, keepdim=True))
    return d.scatter_add_(2, tok, part)


def _plain_prefer(s):
    c = s["c"]
    lp, p, tok, live = _plain_score(s["logits"], s["tokens"], s["lengths"])
    ratio = lp - s["ref"]
    there = (s["chosen"] >= 0) & (s["rejected"] >= 0)
    a, b = s["chosen"].clamp(min=0).long(), s["rejected"].clamp(min=0).long()
    margin = torch.where(there, BETA * (ratio.gather(1, a) - ratio.gather(1, b)), 0.0)
    # -log sigmoid(z) = log(1 + exp(-z)), without overflow
    soft = torch.log1p(torch.exp(-margin.abs()))
    pos, neg = soft + (-margin).clamp(min=0), soft + margin.clamp(min=0)
    eps = c["smoothing"]
    pairs = there.sum().clamp(min=1)
    loss = torch.where(there, (1 - eps) * pos + eps * neg, 0.0).sum() / pairs
    sig = 1 / (1 + torch.exp(-margin))
    w = torch.where(there, BETA * (eps * sig - (1 - eps) * (1 - sig)) / pairs, 0.0)
    g = torch.zeros_like(lp).scatter_add_(1, a, w).scatter_add_(1, b, -w).float()
    return loss.float(), margin.float(), _plain_gradient(p, tok, live, g).to(s["logits"].dtype)


def run(state):
    c = state["c"]
    if own:
        return _own(state)
    if c["op"] == "logits":
        return _plain_logits(state)
    if c["op"] == "propose":
        return _plain_propose(state)
    if c["op"] == "score":
        lp, p, tok, live = _plain_score(state["logits"], state["tokens"], state["lengths"])
        if not c["grad"]:
            return lp.float()
        return lp.float(), _plain_gradient(p, tok, live, state["g"]).to(state["logits"].dtype)
    return _plain_prefer(state)


# ---------------------------------------------------------------- the framework's calls

def _own(s):
    fd = _device_api()
    c = s["c"]
    if c["op"] == "logits":
        return fd.adapter_logits(s["hidden"], s["weight"], s["adapter_ids"], s["lora_a"], s["lora_b"], s["scales"],
                                 out_dtype=DTYPES[c["out"]])
    if c["op"] == "propose":
        return fd.propose(s["logits"], c["k"], order=c["order"])
    if c["op"] == "score":
        if not c["grad"]:
            return fd.sequence_logp(s["logits"], s["tokens"], s["lengths"])
        x = s["logits"].detach().requires_grad_()
        lp = fd.sequence_logp(x, s["tokens"], s["lengths"])
        return lp.detach(), torch.autograd.grad(lp, x, s["g"])[0]
    x = s["logits"].detach().requires_grad_()
    loss, margin = fd.preference_loss(x, s["tokens"], s["lengths"], s["ref"], s["chosen"], s["rejected"], beta=BETA,
                                      label_smoothing=c["smoothing"])
    return loss.detach(), margin, torch.autograd.grad(loss, x)[0]


# ---------------------------------------------------------------- what a pass cannot do without

def _size(name):
    return torch.empty((), dtype=DTYPES[name]).element_size()


def work(case):
    c = case
    n, L, V, b = c["n"], c["L"], c["V"], _size(c["dtype"])
    if c["op"] == "logits":
        D, r = c["D"], c["r"]
        used, rows = min(c["G"], n), n * L
        return dict(bytes=b * (rows * D + V * D + used * r * (D + V)) + 8 * n + rows * V * _size(c["out"]),
                    flops=2 * rows * (V * D + r * D + r * V))
    if c["op"] == "propose":
        return dict(bytes=n * L * (V * b + 8 * c["k"]), flops=4 * n * L * V)
    C = c["C"]
    read = n * L * V * b + 4 * n * C * (L + 1)
    if c["op"] == "score":
        # scores out; with the gradient also its upstream in and the logits' gradient out
        return dict(bytes=read + 4 * n * C + (4 * n * C + n * L * V * b if c["grad"] else 0),
                    flops=(7 if c["grad"] else 4) * n * L * V)
    return dict(bytes=read + 4 * n * C + 12 * n * c["P"] + 4 + n * L * V * b, flops=7 * n * L * V)


# ---------------------------------------------------------------- 64 bits, from the definitions

def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]
    if c["op"] == "logits":
        if c["n"] * c["L"] * c["V"] > 700000000:
            return None
        out = torch.empty((c["n"], c["L"], c["V"]), dtype=torch.float64, device="cuda")
        w = s["weight"].double()
        for i, a in enumerate(s["adapter_ids"].tolist()):
            h = s["hidden"][i].double()
            torch.matmul(h, w.T, out=out[i])
            if a >= 0:
                out[i] += float(s["scales"][a]) * ((h @ s["lora_a"][a].double().T) @ s["lora_b"][a].double().T)
        return out
    logp = torch.empty(s["logits"].shape, dtype=torch.float64, device="cuda")
    for i in range(c["n"]):
        logp[i] = torch.log_softmax(s["logits"][i].double(), -1)
    if c["op"] == "propose":
        ids, lp = [], []
        for i in range(c["n"]):
            v, at = torch.sort(logp[i], dim=-1, descending=True, stable=True)
            v, at = v[:, :c["k"]].clone(), at[:, :c["k"]].clone()
            at[v == float("-inf")] = 1 << 40
            if c["order"] == "id":
                at, by = torch.sort(at, dim=-1, stable=True)
                v = v.gather(-1, by)
            lp.append(torch.where(v == float("-inf"), -FLT_MAX, v))
            ids.append(at)
        return None, torch.stack(lp)
    x = logp.requires_grad_()
    upto = torch.arange(c["L"], device="cuda")[None, None, :] < s["lengths"][:, :, None]
    at = torch.where(upto, s["tokens"], 0).long()
    n, L, C = c["n"], c["L"], c["C"]
    each = x[torch.arange(n, device="cuda")[:, None, None], torch.arange(L, device="cuda")[None, None, :], at]
    lp = (each * upto).sum(-1)
    if c["op"] == "score":
        if not c["grad"]:
            return lp.detach()
        d = torch.autograd.grad(lp, x, s["g"].double())[0]
        return lp.detach(), d - x.detach().exp() * d.sum(-1, keepdim=True)
    losses, margins = [], []
    for i in range(n):
        diff = (lp[i] - s["ref"][i].double())
        there = (s["chosen"][i] >= 0) & (s["rejected"][i] >= 0)
        z = BETA * (diff[s["chosen"][i].clamp(min=0).long()] - diff[s["rejected"][i].clamp(min=0).long()])
        e = c["smoothing"]
        one = (1 - e) * torch.nn.functional.softplus(-z) + e * torch.nn.functional.softplus(z)
        losses.append(one[there])
        margins.append(torch.where(there, z.detach(), 0.0))
    kept = torch.cat(losses)
    loss = kept.sum() / max(1, kept.numel())
    if not kept.numel():
        return loss.detach(), torch.stack(margins), torch.zeros_like(logp)
    d = torch.autograd.grad(loss, x)[0]
    return loss.detach(), torch.stack(margins), d - x.detach().exp() * d.sum(-1, keepdim=True)

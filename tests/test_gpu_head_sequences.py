"""Calls of the model-side operators one behind the other, on streams and
memory that they share."""
import torch
import pytest

from test_gpu_head_ops import make_candidates, make_head, make_logits, make_pairs

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fd(built):
    import flashtrie_device
    return flashtrie_device


def test_direct_calls_on_one_workspace(fd):
    """An adapter for every token (the form whose low-rank part a kernel of its
    own leaves in the workspace): calls that follow one another on the same
    memory, each with other values, give what each gives alone."""
    heads = [make_head(37, 1, 4000, 128, 16, 40, torch.float16, seed=s) for s in range(4)]
    alone = []
    for h, w, ids, a, b, s in heads:
        alone.append(fd.adapter_logits(h, w, ids, a, b, s))
        torch.cuda.synchronize()
    for _ in range(10):
        got = [fd.adapter_logits(h, w, ids, a, b, s) for h, w, ids, a, b, s in heads]
        assert all(torch.equal(p, q) for p, q in zip(alone, got))


@pytest.mark.parametrize("what", ["adapter_logits", "propose", "sequence_logp", "preference_loss", "gradient"])
def test_inputs_dropped_after_a_call_on_another_stream(fd, what):
    """The caller may drop a call's inputs when it returns, and make new tensors
    of their size, although the call's stream has not come to it yet."""
    n, L, V, C = 2, 3, 50000, 7

    def inputs():
        x = make_logits(n, L, V, torch.float32, seed=1, masked=False)
        toks, lens = make_candidates(n, L, V, C, seed=2)
        return x, toks, lens, torch.randn((n, C), device="cuda") * 0, *make_pairs(n, C, 5, seed=3)

    def call(stream):
        if what == "adapter_logits":
            h, w, ids, a, b, s = make_head(n, L, V, 64, 8, 3, torch.bfloat16, seed=4)
            stream.wait_stream(torch.cuda.current_stream())
            return (fd.adapter_logits(h, w, ids, a, b, s, stream=stream),)
        x, toks, lens, ref, c, r = inputs()
        if what == "gradient":
            x.requires_grad_()
        stream.wait_stream(torch.cuda.current_stream())
        if what == "propose":
            return fd.propose(x, 50, stream=stream)
        if what == "sequence_logp":
            return (fd.sequence_logp(x, toks, lens, stream=stream),)
        loss, margin = fd.preference_loss(x, toks, lens, ref, c, r, stream=stream)
        return (margin,) if what == "preference_loss" else torch.autograd.grad(loss, x)

    want = call(torch.cuda.current_stream())
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100000000)  # some 50 ms
    got = call(side)
    # Every size that an input may have had, several times over.
    new = [torch.full((size,), 1.0, device="cuda")
           for size in (n * L * V, V * 32, 3 * V * 4, n * L * 32, n * C * L, n * C, n * 5, 3) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got)) and len(new) == 32

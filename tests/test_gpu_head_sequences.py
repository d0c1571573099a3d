"""Calls of the model-side operators one behind the other, on streams and
memory that they share."""
import torch
import pytest

from test_gpu_head_ops import make_head

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

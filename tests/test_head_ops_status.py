"""The projection's status word: what the C ABI refuses (no GPU needed), and how
a wait that runs out reaches the caller.  The waits themselves never run out
here: the bit is set by a stand-in for the call."""
import ctypes

import pytest
import torch

from test_head_ops_refusals import INVALID, NULL, P, adapter, fd  # noqa: F401

STATE = -1
PROJECTION = 128


def test_status_refusals(fd):  # noqa: F811
    lib, a = fd._lib(), adapter(fd)
    assert lib.ft_adapter_logits_checked_device(ctypes.byref(a), ctypes.c_void_p(4098), P, 1 << 40, None) == INVALID
    assert b"status" in lib.ft_last_error()
    assert lib.ft_adapter_logits_checked_device(None, None, P, 1 << 40, None) == NULL
    empty = adapter(fd, n=0)
    assert lib.ft_adapter_logits_checked_device(ctypes.byref(empty), None, None, 0, None) == 0


def test_status_word_needs_a_workspace(fd):  # noqa: F811
    import flashtrie
    lib, word = fd._lib(), ctypes.c_void_p()
    assert lib.ft_trie_status_word(None, ctypes.byref(word)) == NULL
    t = flashtrie.Trie()
    t.build(token_rows=[[1, 2], [3]])
    assert lib.ft_trie_status_word(ctypes.c_void_p(t.ft_handle()), ctypes.byref(word)) == STATE
    assert lib.ft_trie_status_word(ctypes.c_void_p(t.ft_handle()), None) == NULL
    assert word.value is None


@pytest.mark.gpu
@pytest.mark.parametrize("n,L,G", [(1, 5, 1), (6, 20, 3), (40, 1, 40)])
def test_status_stays_clear(fd, n, L, G):  # noqa: F811
    from test_gpu_head_ops import make_head
    h, w, ids, a, b, s = make_head(n, L, 500, 64, 8, G, torch.bfloat16, seed=1)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = fd.adapter_logits(h, w, ids, a, b, s, status=status)
    assert torch.equal(out, fd.adapter_logits(h, w, ids, a, b, s)) and int(status) == 0
    for bad in (status.long(), torch.zeros(2, dtype=torch.int32, device="cuda"), status[0]):
        with pytest.raises(ValueError):
            fd.adapter_logits(h, w, ids, a, b, s, status=bad)


class _SetsBit:
    """The library, with a projection that reports a wait that ran out."""

    def __init__(self, lib):
        self.lib, self.runtime = lib, ctypes.CDLL("libcudart.so.12")

    def __getattr__(self, name):
        return getattr(self.lib, name)

    def ft_adapter_logits_checked_device(self, args, status, *rest):
        rc = self.lib.ft_adapter_logits_checked_device(args, status, *rest)
        torch.cuda.synchronize()
        bit = ctypes.c_uint32(PROJECTION)
        assert self.runtime.cudaMemcpy(status, ctypes.byref(bit), ctypes.c_size_t(4), 1) == 0
        return rc


@pytest.mark.gpu
def test_a_wait_that_ran_out_reaches_the_caller(fd, monkeypatch):  # noqa: F811
    import flashtrie
    from test_gpu_head_ops import make_head
    t = flashtrie.Trie()
    t.build(token_rows=[[1, 2], [3]])
    t.init_tbs_gpu(1, max_num_topk=8, max_num_outpos=4, max_num_out_beams=4)
    h, w, ids, a, b, s = make_head(1, 4, 50, 64, 8, 2, torch.bfloat16, seed=1)
    beams = torch.full((1, 4), 4, dtype=torch.int32, device="cuda")

    def search(check):
        return fd.bs_tbs_hidden(t, beams, h, w, 8, -10.0, -40.0, 1.0, False, ids, a, b, s, check=check)

    search(True)
    assert fd.device_status(t) == 0
    with monkeypatch.context() as m:
        m.setattr(fd, "_LIB", _SetsBit(fd._lib()))
        with pytest.raises(RuntimeError, match="0x80"):
            search(True)
        search(False)
        assert fd.device_status(t) == PROJECTION
    search(True)

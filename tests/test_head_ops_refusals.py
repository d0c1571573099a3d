"""What the C ABI of the model-side operators refuses, before anything is
launched (no GPU needed), and the workspaces it asks for."""
import ctypes
import types

import pytest
import torch


@pytest.fixture(scope="module")
def fd(built):
    import flashtrie_device
    flashtrie_device._lib()
    return flashtrie_device


INVALID, NULL = -20, -2
P = ctypes.c_void_p(4096)  # never dereferenced: every call here is refused on the host


def adapter(fd, **kw):
    v = dict(n=2, num_outpos=3, vocab=100, dim=64, rank=8, num_adapters=4, dtype=1, out_dtype=1, hidden=P, weight=P,
             adapter_ids=P, lora_a=P, lora_b=P, scale=None, out=P)
    v.update(kw)
    return fd._AdapterArgs(**v)


def propose(fd, **kw):
    v = dict(rows=4, vocab=100, topk=10, dtype=0, order=0, logits=P, topk_id=P, topk_logp=P)
    v.update(kw)
    return fd._ProposeArgs(**v)


def sequence(fd, **kw):
    v = dict(n=2, num_outpos=3, vocab=100, candidates=5, dtype=0, logits=P, tokens=P, lengths=P, stats=P, logp=P,
             grad_logits=P)
    v.update(kw)
    return fd._SequenceArgs(**v)


def preference(fd, **kw):
    v = dict(pairs=4, mean=1, beta=0.1, label_smoothing=0.0, ref_logp=P, chosen=P, rejected=P, margin=P, loss=P,
             grad=P, factor=P)
    v.update(kw)
    return fd._PreferenceArgs(**v)


def size(fd, name, args):
    out = ctypes.c_uint64(0)
    rc = getattr(fd._lib(), "ft_%s_workspace" % name)(ctypes.byref(args), ctypes.byref(out))
    return rc, out.value


@pytest.mark.parametrize("bad", [dict(dtype=0, out_dtype=0), dict(dtype=7), dict(out_dtype=2), dict(out_dtype=9),
                                 dict(num_outpos=0), dict(vocab=0), dict(dim=0), dict(dim=60), dict(rank=0),
                                 dict(rank=12), dict(rank=264), dict(num_adapters=65537),
                                 dict(n=0xFFFFFFFF, num_outpos=0xFFFFFFFF), dict(vocab=0xFFFFFFFF)])
def test_adapter_shapes_refused(fd, bad):
    a = adapter(fd, **bad)
    assert size(fd, "adapter_logits", a)[0] == INVALID
    assert fd._lib().ft_adapter_logits_device(ctypes.byref(a), P, 1 << 40, None) == INVALID
    assert b"adapter_logits" in fd._lib().ft_last_error()


@pytest.mark.parametrize("bad", [dict(hidden=None), dict(weight=None), dict(out=None), dict(adapter_ids=None),
                                 dict(lora_a=None), dict(lora_b=None)])
def test_adapter_null_refused(fd, bad):
    a = adapter(fd, **bad)
    assert fd._lib().ft_adapter_logits_device(ctypes.byref(a), P, 1 << 40, None) == NULL


@pytest.mark.parametrize("bad", [dict(hidden=4098), dict(weight=4104), dict(lora_a=4098), dict(lora_b=4104), dict(out=4098)])
def test_adapter_unaligned_refused(fd, bad):
    a = adapter(fd, **{k: ctypes.c_void_p(v) for k, v in bad.items()})
    assert fd._lib().ft_adapter_logits_device(ctypes.byref(a), P, 1 << 40, None) == INVALID


def test_adapter_workspace_refused_and_empty_batch(fd):
    a = adapter(fd)
    rc, need = size(fd, "adapter_logits", a)
    assert rc == 0 and need > 0
    for ws, have in ((P, need - 1), (None, need), (ctypes.c_void_p(4097), need)):
        assert fd._lib().ft_adapter_logits_device(ctypes.byref(a), ws, have, None) == INVALID
    empty = adapter(fd, n=0)
    assert fd._lib().ft_adapter_logits_device(ctypes.byref(empty), None, 0, None) == 0


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(vocab=0), dict(vocab=0xFFFFFFFF), dict(topk=0), dict(topk=8193),
                                 dict(order=2), dict(order=-1), dict(rows=1 << 31), dict(logits=ctypes.c_void_p(4098))])
def test_propose_refused(fd, bad):
    a = propose(fd, **bad)
    assert fd._lib().ft_propose_device(ctypes.byref(a), P, 1 << 40, None) == INVALID
    assert b"propose" in fd._lib().ft_last_error()


@pytest.mark.parametrize("bad", [dict(logits=None), dict(topk_id=None), dict(topk_logp=None)])
def test_propose_null_refused(fd, bad):
    a = propose(fd, **bad)
    assert fd._lib().ft_propose_device(ctypes.byref(a), P, 1 << 40, None) == NULL


def test_propose_empty_batch(fd):
    a = propose(fd, rows=0, logits=None)
    assert fd._lib().ft_propose_device(ctypes.byref(a), None, 0, None) == 0


@pytest.mark.parametrize("bad", [dict(dtype=-1), dict(num_outpos=0), dict(vocab=0), dict(candidates=0),
                                 dict(candidates=8193), dict(n=0x80000000, num_outpos=1),
                                 dict(n=0x40000000, num_outpos=2), dict(n=0x7FFFFFFF, num_outpos=1, candidates=33)])
def test_sequence_shapes_refused(fd, bad):
    a = sequence(fd, **bad)
    lib = fd._lib()
    assert size(fd, "sequence_logp", a)[0] == INVALID
    assert size(fd, "preference_loss", a)[0] == INVALID
    assert lib.ft_sequence_logp_device(ctypes.byref(a), P, 1 << 60, None) == INVALID
    assert lib.ft_sequence_grad_device(ctypes.byref(a), P, None, None, P, 1 << 60, None) == INVALID
    assert lib.ft_preference_loss_device(ctypes.byref(a), ctypes.byref(preference(fd)), P, 1 << 60, None) == INVALID


@pytest.mark.parametrize("bad", [dict(logits=None), dict(tokens=None), dict(lengths=None), dict(stats=None)])
def test_sequence_null_refused(fd, bad):
    a = sequence(fd, **bad)
    lib = fd._lib()
    assert lib.ft_sequence_logp_device(ctypes.byref(a), P, 1 << 40, None) == NULL
    assert lib.ft_sequence_grad_device(ctypes.byref(a), P, None, None, P, 1 << 40, None) == NULL
    assert lib.ft_preference_loss_device(ctypes.byref(a), ctypes.byref(preference(fd)), P, 1 << 40, None) == NULL


def test_sequence_own_outputs_refused(fd):
    lib = fd._lib()
    assert lib.ft_sequence_logp_device(ctypes.byref(sequence(fd, logp=None)), P, 1 << 40, None) == NULL
    assert lib.ft_sequence_grad_device(ctypes.byref(sequence(fd, grad_logits=None)), P, None, None, P, 1 << 40,
                                       None) == NULL
    assert lib.ft_sequence_grad_device(ctypes.byref(sequence(fd)), None, None, None, P, 1 << 40, None) == NULL
    odd = sequence(fd, logits=ctypes.c_void_p(4098))
    assert lib.ft_sequence_logp_device(ctypes.byref(odd), P, 1 << 40, None) == INVALID


@pytest.mark.parametrize("bad", ["ref_logp", "chosen", "rejected", "margin", "loss", "grad", "factor"])
def test_preference_null_refused(fd, bad):
    p = preference(fd, **{bad: None})
    assert fd._lib().ft_preference_loss_device(ctypes.byref(sequence(fd)), ctypes.byref(p), P, 1 << 40, None) == NULL


def test_preference_too_many_pairs_refused(fd):
    p = preference(fd, pairs=1 << 30)
    assert fd._lib().ft_preference_loss_device(ctypes.byref(sequence(fd)), ctypes.byref(p), P, 1 << 40, None) == INVALID


@pytest.mark.parametrize("eps", [-0.1, 1.5, float("nan")])
def test_preference_smoothing_refused(fd, eps):
    p = preference(fd, label_smoothing=eps)
    assert fd._lib().ft_preference_loss_device(ctypes.byref(sequence(fd)), ctypes.byref(p), P, 1 << 40, None) == INVALID


@pytest.mark.parametrize("beta", [float("inf"), float("-inf"), float("nan")])
def test_preference_beta_refused(fd, beta):
    p = preference(fd, beta=beta)
    assert fd._lib().ft_preference_loss_device(ctypes.byref(sequence(fd)), ctypes.byref(p), P, 1 << 40, None) == INVALID


def test_stream_of_another_device_refused(fd):
    stream = types.SimpleNamespace(device_index=1)
    with pytest.raises(ValueError, match="stream"):
        fd._On(torch.device("cuda", 0), stream)


def test_sequence_workspaces(fd):
    a = sequence(fd)
    lib = fd._lib()
    for name, call in (("sequence_logp", lambda ws, have: lib.ft_sequence_logp_device(
            ctypes.byref(a), ws, have, None)),
                       ("preference_loss", lambda ws, have: lib.ft_preference_loss_device(
                                 ctypes.byref(a), ctypes.byref(preference(fd)), ws, have, None))):
        rc, need = size(fd, name, a)
        assert rc == 0 and need > 0
        assert call(P, 8) == INVALID
        assert call(None, need) == NULL
        assert call(ctypes.c_void_p(4097), need) == INVALID


def test_null_arguments(fd):
    lib, out = fd._lib(), ctypes.c_uint64(0)
    for name in ("adapter_logits", "propose", "sequence_logp"):
        assert getattr(lib, "ft_%s_workspace" % name)(None, ctypes.byref(out)) == NULL
        assert getattr(lib, "ft_%s_device" % name)(None, None, 0, None) == NULL
    assert lib.ft_preference_loss_device(ctypes.byref(sequence(fd)), None, None, 0, None) == NULL


def test_cpu_tensors_refused(fd):
    import torch
    x = torch.zeros((1, 2, 16), dtype=torch.bfloat16)
    ints = torch.zeros((1, 3), dtype=torch.int32)
    with pytest.raises(TypeError):
        fd.adapter_logits(x, torch.zeros((5, 16), dtype=torch.bfloat16))
    with pytest.raises(TypeError):
        fd.propose(x, 3)
    with pytest.raises(TypeError):
        fd.sequence_logp(x, torch.zeros((1, 3, 2), dtype=torch.int32), ints)
    with pytest.raises(TypeError):
        fd.preference_loss(x, torch.zeros((1, 3, 2), dtype=torch.int32), ints, ints.float(), ints, ints)

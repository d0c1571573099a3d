"""Trie-constrained beam search on inputs that already live in device memory.

For callers whose proposals come out of a model on the GPU (the top-k of the
logits at each position): the search reads them where they are and writes
its results to device tensors, on the caller's CUDA stream, with no host
copy in between.  This is the C-ABI entry point `ft_tbs_batch_device`
(include/flashtrie_b200.h); the reference has no counterpart (its
`bs_tbs_gpu` always stages host lists, tools/bindings.cpp:71-119).

    import torch, flashtrie, flashtrie_device as fd
    trie = flashtrie.Trie(); trie.load("trie.bin")
    trie.init_tbs_gpu(64, max_num_topk=1000, max_num_outpos=20, max_num_out_beams=1000)
    out = fd.bs_tbs_device(trie, beams, topk_id, topk_logp, -10.0, -40.0, 5.0, False)
    sents, lpns = fd.to_lists(out)        # host lists, only when needed
    ids = fd.lookup(trie, tokens, offsets)  # key ids of token sequences on the device
    toks, lens = fd.reverse_lookup(trie, ids, max_len=20)  # and back

Inputs (contiguous, on one CUDA device): beams int32 [n, L]; topk_id int32
[n, L, K] (token ids, read as unsigned); topk_logp float32 [n, L, K].  Rows
need not be sorted by id.  The search runs on `stream` (default: the current
stream); inputs written on another stream must be ordered before it by the
caller (an event, or stream.wait_stream), and the outputs are allocated on
`stream`.  Outputs: count int32 [n]; logp_norm float64
[n, cap] ascending; lengths int32 [n, cap]; tokens int32 [n, cap, L], beam j
of request i in tokens[i, j, :lengths[i, j]]; with key_ids=True also key ids
int32 [n, cap] (LoudsTrie::lookup's id of each result, read as unsigned).

The steps between a model and the search, on the same tensors and with the
same stream rules:

    logits = fd.adapter_logits(hidden, weight, adapter_ids, lora_a, lora_b)  # [n, L, V]
    topk_id, topk_logp = fd.propose(logits, 1000)            # the search's proposals
    out = fd.bs_tbs_hidden(trie, beams, hidden, weight, 1000, -10.0, -40.0, 5.0, False)  # both, and the search
    count, lpn, lens, toks = out
    ref = fd.sequence_logp(ref_logits, toks, lens)           # scores of the results, differentiable
    loss, margin = fd.preference_loss(logits, toks, lens, ref, chosen, rejected)  # differentiable
"""
import ctypes
import functools
import math
import os

import torch
from torch.autograd.function import once_differentiable

_HERE = os.path.dirname(os.path.abspath(__file__))
_LIB = None


class _Params(ctypes.Structure):
    _fields_ = [("token_logp_threshold", ctypes.c_float), ("reserved", ctypes.c_float),
                ("sent_logp_threshold", ctypes.c_double), ("length_norm", ctypes.c_double),
                ("early_exit", ctypes.c_int32), ("reserved2", ctypes.c_int32)]


class _Batch(ctypes.Structure):
    _fields_ = [("n", ctypes.c_uint32), ("num_outpos", ctypes.c_uint32), ("topk", ctypes.c_uint32),
                ("out_capacity", ctypes.c_uint32)] + [(f, ctypes.c_void_p) for f in
                                                      ("beams", "topk_id", "topk_logp", "out_count", "out_lpn",
                                                       "out_len", "out_tok", "out_key")]


class _AdapterArgs(ctypes.Structure):
    _fields_ = [(f, ctypes.c_uint32) for f in ("n", "num_outpos", "vocab", "dim", "rank", "num_adapters")] + \
        [("dtype", ctypes.c_int32), ("out_dtype", ctypes.c_int32)] + \
        [(f, ctypes.c_void_p) for f in ("hidden", "weight", "adapter_ids", "lora_a", "lora_b", "scale", "out")]


class _ProposeArgs(ctypes.Structure):
    _fields_ = [("rows", ctypes.c_uint64), ("vocab", ctypes.c_uint32), ("topk", ctypes.c_uint32),
                ("dtype", ctypes.c_int32), ("order", ctypes.c_int32)] + \
        [(f, ctypes.c_void_p) for f in ("logits", "topk_id", "topk_logp")]


class _SequenceArgs(ctypes.Structure):
    _fields_ = [(f, ctypes.c_uint32) for f in ("n", "num_outpos", "vocab", "candidates")] + \
        [("dtype", ctypes.c_int32), ("reserved", ctypes.c_int32)] + \
        [(f, ctypes.c_void_p) for f in ("logits", "tokens", "lengths", "stats", "logp", "grad_logits")]


class _PreferenceArgs(ctypes.Structure):
    _fields_ = [("pairs", ctypes.c_uint32), ("mean", ctypes.c_int32), ("beta", ctypes.c_float),
                ("label_smoothing", ctypes.c_float)] + \
        [(f, ctypes.c_void_p) for f in ("ref_logp", "chosen", "rejected", "margin", "loss", "grad", "factor")]


# FT_DTYPE_* of include/flashtrie_b200.h.
_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _lib():
    global _LIB
    if _LIB is None:
        lib = ctypes.CDLL(os.path.join(_HERE, "libftcore.so"))
        lib.ft_tbs_batch_device.argtypes = [ctypes.c_void_p, ctypes.POINTER(_Batch), ctypes.POINTER(_Params),
                                            ctypes.c_void_p]
        lib.ft_tbs_batch_device.restype = ctypes.c_int
        lib.ft_lookup_batch_device.argtypes = [ctypes.c_void_p, ctypes.c_uint32, ctypes.c_void_p, ctypes.c_void_p,
                                               ctypes.c_uint64, ctypes.c_void_p, ctypes.c_void_p]
        lib.ft_lookup_batch_device.restype = ctypes.c_int
        lib.ft_reverse_lookup_batch_device.argtypes = [ctypes.c_void_p, ctypes.c_uint32, ctypes.c_void_p,
                                                       ctypes.c_uint32, ctypes.c_void_p, ctypes.c_void_p,
                                                       ctypes.c_void_p]
        lib.ft_reverse_lookup_batch_device.restype = ctypes.c_int
        lib.ft_trie_device_status.argtypes = [ctypes.c_void_p, ctypes.POINTER(ctypes.c_uint32)]
        lib.ft_trie_device_status.restype = ctypes.c_int
        lib.ft_trie_status_word.argtypes = [ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p)]
        lib.ft_trie_status_word.restype = ctypes.c_int
        lib.ft_last_error.restype = ctypes.c_char_p
        u64p, vp, u64 = ctypes.POINTER(ctypes.c_uint64), ctypes.c_void_p, ctypes.c_uint64
        for name, args in (("adapter_logits", _AdapterArgs), ("propose", _ProposeArgs),
                           ("sequence_logp", _SequenceArgs)):
            size, call = getattr(lib, "ft_%s_workspace" % name), getattr(lib, "ft_%s_device" % name)
            size.argtypes = [ctypes.POINTER(args), u64p]
            call.argtypes = [ctypes.POINTER(args), vp, u64, vp]
        lib.ft_adapter_logits_checked_device.argtypes = [ctypes.POINTER(_AdapterArgs), vp, vp, u64, vp]
        lib.ft_sequence_grad_device.argtypes = [ctypes.POINTER(_SequenceArgs), vp, vp, vp, vp, u64, vp]
        lib.ft_preference_loss_workspace.argtypes = [ctypes.POINTER(_SequenceArgs), u64p]
        lib.ft_preference_loss_device.argtypes = [ctypes.POINTER(_SequenceArgs), ctypes.POINTER(_PreferenceArgs), vp,
                                                  u64, vp]
        _LIB = lib
    return _LIB


def _check(rc):
    if rc != 0:
        raise RuntimeError(_lib().ft_last_error().decode())


def _want(t, name, dtype, ndim, device):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError("%s must be a CUDA tensor" % name)
    if t.dtype != dtype or t.dim() != ndim or not t.is_contiguous():
        raise ValueError("%s must be a contiguous %s tensor with %d dimensions" % (name, dtype, ndim))
    if device is not None and t.get_device() != device.index:
        raise ValueError("%s is on %s, expected %s" % (name, t.device, device))


def device_status(trie):
    """Synchronises the device and returns (and clears) the status bits of the
    device-resident searches since the last call (0: all searches passed their
    self-checks)."""
    st = ctypes.c_uint32(0)
    _check(_lib().ft_trie_device_status(ctypes.c_void_p(trie.ft_handle()), ctypes.byref(st)))
    return st.value


def bs_tbs_device(trie, beams, topk_id, topk_logp, token_logp_threshold, sents_logp_threshold, length_norm,
                  early_exit, capacity=None, stream=None, check=True, key_ids=False):
    """Searches n requests whose inputs are CUDA tensors; returns
    (count, logp_norm, lengths, tokens[, keys]) as CUDA tensors on the same
    device (keys with key_ids=True).

    capacity: result slots per request (>= every final beam width); default
    beams[:, -1].max(), which reads one value back from the device.
    stream: a torch.cuda.Stream (default: the current stream of the device).
    check: synchronise after the search and raise if a self-check failed or a
    request exceeded the workspace; with check=False the call is asynchronous
    and device_status() reports later."""
    _want(beams, "beams", torch.int32, 2, None)
    dev = beams.device
    _want(topk_id, "topk_id", torch.int32, 3, dev)
    _want(topk_logp, "topk_logp", torch.float32, 3, dev)
    n, L = beams.shape
    if topk_id.shape[:2] != (n, L) or topk_logp.shape != topk_id.shape:
        raise ValueError("topk_id and topk_logp must be [n, L, K] with n, L matching beams")
    K = topk_id.shape[2]
    if capacity is None:
        capacity = int(beams[:, -1].max().item()) if n and L else 1
    capacity = max(int(capacity), 1)
    if stream is None:
        stream = torch.cuda.current_stream(dev)
    # The outputs are allocated and filled on the search's stream, so the
    # fills come before the search writes them whatever stream is current.
    with torch.cuda.stream(stream):
        count = torch.zeros(n, dtype=torch.int32, device=dev)
        lpn = torch.empty((n, capacity), dtype=torch.float64, device=dev)
        lens = torch.zeros((n, capacity), dtype=torch.int32, device=dev)
        toks = torch.empty((n, capacity, max(L, 1)), dtype=torch.int32, device=dev)
        keys = torch.full((n, capacity), -1, dtype=torch.int32, device=dev) if key_ids else None
    out = (count, lpn, lens, toks) + ((keys,) if key_ids else ())
    if n == 0:
        return out
    b = _Batch(n, L, K, capacity, beams.data_ptr(), topk_id.data_ptr(), topk_logp.data_ptr(), count.data_ptr(),
               lpn.data_ptr(), lens.data_ptr(), toks.data_ptr(), keys.data_ptr() if key_ids else None)
    prm = _Params(float(token_logp_threshold), 0.0, float(sents_logp_threshold), float(length_norm),
                  int(bool(early_exit)), 0)
    with torch.cuda.device(dev):
        _check(_lib().ft_tbs_batch_device(ctypes.c_void_p(trie.ft_handle()), ctypes.byref(b), ctypes.byref(prm),
                                          ctypes.c_void_p(stream.cuda_stream)))
    if check:
        st = device_status(trie)
        if st:
            raise RuntimeError("device search failed its self-checks or exceeded the workspace (status 0x%x)" % st)
    return out


def lookup(trie, tokens, offsets, stream=None, check=True):
    """Key ids of n token sequences on the device: LoudsTrie::lookup for a
    batch (C ABI ft_lookup_batch_device).  tokens: int32 CUDA tensor [T]
    (ids read as unsigned); offsets: int64 CUDA tensor [n + 1], key i being
    tokens[offsets[i]:offsets[i + 1]].  Returns an int32 tensor [n] of key
    ids (the ids key_ids=True reports; read as unsigned), -1 where the
    sequence is not a key.  check: synchronise and raise if the kernel
    reported bad offsets or an inconsistent trie."""
    _want(tokens, "tokens", torch.int32, 1, None)
    dev = tokens.device
    _want(offsets, "offsets", torch.int64, 1, dev)
    n = offsets.numel() - 1
    if n < 0:
        raise ValueError("offsets must have n + 1 >= 1 entries")
    if stream is None:
        stream = torch.cuda.current_stream(dev)
    with torch.cuda.stream(stream):
        out = torch.empty(n, dtype=torch.int32, device=dev)
    if n == 0:
        return out
    with torch.cuda.device(dev):
        _check(_lib().ft_lookup_batch_device(ctypes.c_void_p(trie.ft_handle()), n, ctypes.c_void_p(tokens.data_ptr()),
                                             ctypes.c_void_p(offsets.data_ptr()), tokens.numel(),
                                             ctypes.c_void_p(out.data_ptr()), ctypes.c_void_p(stream.cuda_stream)))
    if check:
        st = device_status(trie)
        if st:
            raise RuntimeError("device lookup reported bad offsets or an inconsistent trie (status 0x%x)" % st)
    return out


def reverse_lookup(trie, ids, max_len, stream=None, check=True):
    """Token sequences of key ids on the device: LoudsTrie::reverse_lookup
    for a batch (C ABI ft_reverse_lookup_batch_device).  ids: int32 CUDA
    tensor [n] (read as unsigned).  Returns (tokens int32 [n, max_len],
    lengths int32 [n]): key i is tokens[i, :lengths[i]] when lengths[i] <=
    max_len (longer keys report their length and write no tokens); -1 marks
    an id that is not a key id.  The first call derives the trie's parent
    links on the device once."""
    _want(ids, "ids", torch.int32, 1, None)
    dev = ids.device
    n = ids.numel()
    max_len = int(max_len)
    if max_len < 0:
        raise ValueError("max_len must be >= 0")
    if stream is None:
        stream = torch.cuda.current_stream(dev)
    with torch.cuda.stream(stream):
        toks = torch.zeros((n, max(max_len, 1)), dtype=torch.int32, device=dev)
        lens = torch.empty(n, dtype=torch.int32, device=dev)
    if n == 0:
        return toks[:, :max_len], lens
    with torch.cuda.device(dev):
        _check(_lib().ft_reverse_lookup_batch_device(ctypes.c_void_p(trie.ft_handle()), n,
                                                     ctypes.c_void_p(ids.data_ptr()), max_len,
                                                     ctypes.c_void_p(toks.data_ptr()), ctypes.c_void_p(lens.data_ptr()),
                                                     ctypes.c_void_p(stream.cuda_stream)))
    if check:
        st = device_status(trie)
        if st:
            raise RuntimeError("device reverse lookup found an inconsistent trie (status 0x%x)" % st)
    return toks[:, :max_len], lens


def to_lists(out):
    """(count, logp_norm, lengths, tokens[, keys]) -> (sentences, logp_norms
    [, key_ids]) as host lists in the layout bs_tbs_gpu returns."""
    host = [t.cpu() for t in out]
    count, lpn, lens, toks = host[:4]
    sents, lpns, keys = [], [], []
    for i in range(count.shape[0]):
        c = int(count[i])
        sents.append([(toks[i, j, :int(lens[i, j])].numpy().view("uint32")).tolist() for j in range(c)])
        lpns.append(lpn[i, :c].tolist())
        if len(host) > 4:
            keys.append(host[4][i, :c].numpy().view("uint32").tolist())
    return (sents, lpns, keys) if len(host) > 4 else (sents, lpns)


def _want_floating(t, name, ndim, device, dtypes):
    """_want for a tensor of one of several floating types."""
    dtype = t.dtype if isinstance(t, torch.Tensor) and t.dtype in dtypes else dtypes[0]
    _want(t, name, dtype, ndim, device)


def _no_gradient(what, **tensors):
    if torch.is_grad_enabled():
        for name, t in tensors.items():
            if t is not None and t.requires_grad:
                raise ValueError("%s has no gradient: detach %s or call it under torch.no_grad()" % (what, name))


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(call, args, *shape):
    """Bytes that C ABI call `call` asks for at a shape (the leading fields of
    its argument struct)."""
    need = ctypes.c_uint64(0)
    _check(getattr(_lib(), call)(ctypes.byref(args(*shape)), ctypes.byref(need)))
    return need.value


def _workspace(device, *what):
    """(tensor, pointer, bytes) of a call's workspace, on the current stream."""
    need = _workspace_bytes(*what)
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr(), need


def _raw_stream(device):
    return torch.cuda.current_stream(device.index).cuda_stream


class _On:
    """The call's device and stream made current, where they are not already.
    Inputs are noted as in use on a stream that is not the current one: their
    memory, if the caller drops them, waits for what that stream has to do."""

    def __init__(self, device, stream, *inputs):
        self.inner = []
        if stream is not None and stream.device_index != device.index:
            raise ValueError("stream must be of the tensors' device, cuda:%d" % device.index)
        if torch.cuda.current_device() != device.index:
            self.inner.append(torch.cuda.device(device))
        if stream is not None:
            self.inner.append(torch.cuda.stream(stream))
            if stream != torch.cuda.current_stream(device):
                for t in inputs:
                    if t is not None:
                        t.record_stream(stream)

    def __enter__(self):
        for c in self.inner:
            c.__enter__()

    def __exit__(self, *error):
        for c in reversed(self.inner):
            c.__exit__(*error)


def adapter_logits(hidden, weight, adapter_ids=None, lora_a=None, lora_b=None, scale=None, out_dtype=None, stream=None,
                   status=None):
    """Logits of n requests over the vocabulary, each request with a low-rank
    adapter of its own beside the shared projection (C ABI
    ft_adapter_logits_device):

        out[i] = hidden[i] @ weight.T + scale[a] * (hidden[i] @ lora_a[a].T) @ lora_b[a].T,  a = adapter_ids[i]

    hidden: bfloat16 or float16 [n, L, D]; weight [V, D], lora_a [G, r, D]
    and lora_b [G, V, r] of the same type; adapter_ids int32 [n]; scale
    float32 [G] (default 1).  D and r are multiples of 8, r <= 256.  An id of
    -1 takes the shared projection alone; any other id outside [0, G) makes
    that request's logits NaN.  Without adapter_ids there are no adapters.
    Infinities and NaN in an adapter reach its own requests only; where lora_b
    or the product with lora_a is infinite the logit is NaN or infinite.
    Products are summed in 32 bits and the logits rounded once; the low-rank
    values between the two products may have any size that float32 holds and
    lose 2^-17 at most (2^-26 for float32 logits of bfloat16 operands; float16
    ones 2^-23, or 2^-25 absolute and 2^-17 of the token's largest).  Returns
    [n, L, V] of out_dtype (hidden's type, the default, or float32).  For
    serving: it has no gradient.

    status: an int32 CUDA tensor of one element (or None).  The kernel's waits
    are bounded; where one runs out it sets a bit there and leaves NaN in the
    logits that it has not made.  Nothing clears the bit."""
    if status is not None:
        _want(status, "status", torch.int32, 1, hidden.device if isinstance(hidden, torch.Tensor) else None)
        if status.numel() != 1:
            raise ValueError("status must have one element")
        status = status.data_ptr()
    return _logits(hidden, weight, adapter_ids, lora_a, lora_b, scale, out_dtype, stream, status)


def _logits(hidden, weight, adapter_ids, lora_a, lora_b, scale, out_dtype, stream, status):
    """adapter_logits with the status word's address."""
    _want_floating(hidden, "hidden", 3, None, (torch.bfloat16, torch.float16))
    dev, dt = hidden.device, hidden.dtype
    _want(weight, "weight", dt, 2, dev)
    n, L, D = hidden.shape
    V = weight.shape[0]
    if weight.shape[1] != D:
        raise ValueError("weight must be [V, D] with D = %d, hidden's" % D)
    out_dtype = dt if out_dtype is None else out_dtype
    if out_dtype not in (dt, torch.float32):
        raise ValueError("out_dtype must be hidden's type or torch.float32")
    G = r = 0
    if adapter_ids is None:
        if lora_a is not None or lora_b is not None or scale is not None:
            raise ValueError("lora_a, lora_b and scale need adapter_ids")
    else:
        if lora_a is None or lora_b is None:
            raise ValueError("adapter_ids needs lora_a and lora_b")
        _want(adapter_ids, "adapter_ids", torch.int32, 1, dev)
        _want(lora_a, "lora_a", dt, 3, dev)
        _want(lora_b, "lora_b", dt, 3, dev)
        G, r = lora_a.shape[:2]
        if adapter_ids.shape[0] != n or lora_a.shape[2] != D or tuple(lora_b.shape) != (G, V, r) or G == 0:
            raise ValueError("adapter_ids must be [n], lora_a [G, r, D] and lora_b [G, V, r] with G >= 1")
        if scale is not None:
            _want(scale, "scale", torch.float32, 1, dev)
            if scale.shape[0] != G:
                raise ValueError("scale must have one value per adapter")
    _no_gradient("adapter_logits", hidden=hidden, weight=weight, lora_a=lora_a, lora_b=lora_b, scale=scale)
    if L == 0 or V == 0 or D == 0:
        raise ValueError("L, V and D must be positive")
    shape = (n, L, V, D, r, G, _DTYPE[dt], _DTYPE[out_dtype])
    with _On(dev, stream, hidden, weight, adapter_ids, lora_a, lora_b, scale):
        ws, ws_ptr, ws_bytes = _workspace(dev, "ft_adapter_logits_workspace", _AdapterArgs, *shape)
        out = torch.empty(n, L, V, dtype=out_dtype, device=dev)
        a = _AdapterArgs(*shape, hidden.data_ptr(), weight.data_ptr(), adapter_ids.data_ptr() if G else None,
                         lora_a.data_ptr() if G else None, lora_b.data_ptr() if G else None,
                         scale.data_ptr() if scale is not None else None, out.data_ptr())
        _check(_lib().ft_adapter_logits_checked_device(ctypes.byref(a), status, ws_ptr, ws_bytes, _raw_stream(dev)))
    return out


def propose(logits, k, order="id", stream=None):
    """The search's proposals from logits (C ABI ft_propose_device): per
    position the log-softmax over the vocabulary and its k largest entries,
    equal logits in order of the token id.  logits: float32, bfloat16 or
    float16 [n, L, V].  Returns (topk_id int32 [n, L, k], topk_logp float32
    [n, L, k]), what bs_tbs_device takes.

    order: "id" (ascending token ids, which the search reads without sorting)
    or "logp" (best first).  Logits of -inf are never proposed: a position
    with fewer than k others ends with (-1, -3.4028235e38), entries that no
    search step takes, and a position without a distribution (a NaN or +inf
    among its logits, or -inf alone) holds nothing else.  1 <= k <= 8192; it
    may exceed V.  The outputs have no gradient."""
    _want_floating(logits, "logits", 3, None, (torch.float32, torch.bfloat16, torch.float16))
    dev = logits.device
    n, L, V = logits.shape
    k = int(k)
    if not 1 <= k <= 8192:
        raise ValueError("k must be in [1, 8192]")
    if order not in ("id", "logp"):
        raise ValueError("order must be 'id' or 'logp'")
    if V == 0:
        raise ValueError("the vocabulary is empty")
    _no_gradient("propose", logits=logits)
    shape = (n * L, V, k, _DTYPE[logits.dtype], int(order == "logp"))
    with _On(dev, stream, logits):
        ids = torch.empty(n, L, k, dtype=torch.int32, device=dev)
        lps = torch.empty(n, L, k, dtype=torch.float32, device=dev)
        if n * L:
            ws, ws_ptr, ws_bytes = _workspace(dev, "ft_propose_workspace", _ProposeArgs, *shape)
            a = _ProposeArgs(*shape, logits.data_ptr(), ids.data_ptr(), lps.data_ptr())
            _check(_lib().ft_propose_device(ctypes.byref(a), ws_ptr, ws_bytes, _raw_stream(dev)))
    return ids, lps


def bs_tbs_hidden(trie, beams, hidden, weight, k, token_logp_threshold, sents_logp_threshold, length_norm, early_exit,
                  adapter_ids=None, lora_a=None, lora_b=None, scale=None, logits_dtype=torch.float32, capacity=None,
                  stream=None, check=True, key_ids=False):
    """bs_tbs_device from a model's hidden states: adapter_logits (in
    logits_dtype), the k best proposals of each position, and the search, one
    after the other on `stream`.  hidden [n, L, D] goes with beams [n, L];
    the other arguments and the outputs are those of the three calls.  A wait
    of the projection that ran out is reported as the search's failures are:
    raised with check=True, by device_status() otherwise."""
    _want(beams, "beams", torch.int32, 2, None)
    _want_floating(hidden, "hidden", 3, beams.device, (torch.bfloat16, torch.float16))
    if hidden.shape[:2] != beams.shape:
        raise ValueError("hidden must be [n, L, D] with n, L matching beams")
    word = ctypes.c_void_p()
    if beams.shape[0]:
        _check(_lib().ft_trie_status_word(ctypes.c_void_p(trie.ft_handle()), ctypes.byref(word)))
    logits = _logits(hidden, weight, adapter_ids, lora_a, lora_b, scale, logits_dtype, stream, word)
    topk_id, topk_logp = propose(logits, k, stream=stream)
    del logits
    _On(beams.device, stream, beams)
    return bs_tbs_device(trie, beams, topk_id, topk_logp, token_logp_threshold, sents_logp_threshold, length_norm,
                         early_exit, capacity=capacity, stream=stream, check=check, key_ids=key_ids)


def _sequence_shape(logits, tokens):
    n, L, V = logits.shape
    return n, L, V, tokens.shape[1], _DTYPE[logits.dtype], 0


def _sequence_grad(logits, tokens, lengths, stats, grad, factor, upstream):
    """Gradient of the logits, on the current stream (autograd makes the
    forward call's current). stats, grad, factor, upstream: device pointers."""
    dev = logits.device
    with _On(dev, None):
        out = torch.empty_like(logits)
        if logits.numel() == 0 or tokens.shape[1] == 0:
            return out.zero_()
        shape = _sequence_shape(logits, tokens)
        ws, ws_ptr, ws_bytes = _workspace(dev, "ft_sequence_logp_workspace", _SequenceArgs, *shape)
        a = _SequenceArgs(*shape, logits.data_ptr(), tokens.data_ptr(), lengths.data_ptr(), stats, None, out.data_ptr())
        _check(_lib().ft_sequence_grad_device(ctypes.byref(a), grad, factor, upstream, ws_ptr, ws_bytes,
                                              _raw_stream(dev)))
    return out


def _scores(logits, tokens, lengths):
    """(scores, what the gradient needs beside the inputs)"""
    dev = logits.device
    shape = _sequence_shape(logits, tokens)
    logp = torch.empty(*lengths.shape, dtype=torch.float32, device=dev)
    stats = torch.empty(*shape[:2], 2, dtype=torch.float32, device=dev)
    if logp.numel():
        ws, ws_ptr, ws_bytes = _workspace(dev, "ft_sequence_logp_workspace", _SequenceArgs, *shape)
        a = _SequenceArgs(*shape, logits.data_ptr(), tokens.data_ptr(), lengths.data_ptr(), stats.data_ptr(),
                          logp.data_ptr(), None)
        _check(_lib().ft_sequence_logp_device(ctypes.byref(a), ws_ptr, ws_bytes, _raw_stream(dev)))
    return logp, stats


def _preference(logits, tokens, lengths, ref_logp, chosen, rejected, beta, label_smoothing, mean):
    """(loss, margin, what the gradient needs beside the inputs: the rows'
    statistics, the candidates' gradients and their common factor in one
    tensor)"""
    dev = logits.device
    shape = _sequence_shape(logits, tokens)
    n, L, C = shape[0], shape[1], shape[3]
    margin = torch.empty(*chosen.shape, dtype=torch.float32, device=dev)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    kept = torch.empty(2 * n * L + n * C + 1, dtype=torch.float32, device=dev)
    ws, ws_ptr, ws_bytes = _workspace(dev, "ft_preference_loss_workspace", _SequenceArgs, *shape)
    at = kept.data_ptr()
    a = _SequenceArgs(*shape, logits.data_ptr(), tokens.data_ptr(), lengths.data_ptr(), at, None, None)
    p = _PreferenceArgs(chosen.shape[1], int(mean), beta, label_smoothing, ref_logp.data_ptr(), chosen.data_ptr(),
                        rejected.data_ptr(), margin.data_ptr(), loss.data_ptr(), at + 8 * n * L,
                        at + 8 * n * L + 4 * n * C)
    _check(_lib().ft_preference_loss_device(ctypes.byref(a), ctypes.byref(p), ws_ptr, ws_bytes, _raw_stream(dev)))
    return loss, margin, kept


class _SequenceLogp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, lengths):
        logp, stats = _scores(logits, tokens, lengths)
        ctx.save_for_backward(logits, tokens, lengths, stats)
        return logp

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        logits, tokens, lengths, stats = ctx.saved_tensors
        g = g.contiguous()
        return _sequence_grad(logits, tokens, lengths, stats.data_ptr(), g.data_ptr(), None, None), None, None


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, lengths, *rest):
        loss, margin, kept = _preference(logits, tokens, lengths, *rest)
        ctx.save_for_backward(logits, tokens, lengths, kept)
        ctx.mark_non_differentiable(margin)
        ctx.set_materialize_grads(False)  # the margin's is not looked at
        return loss, margin

    @staticmethod
    @once_differentiable
    def backward(ctx, g, _):
        if g is None:
            return (None,) * 9
        logits, tokens, lengths, kept = ctx.saved_tensors
        n, L, C = logits.shape[0], logits.shape[1], tokens.shape[1]
        at = kept.data_ptr()
        return (_sequence_grad(logits, tokens, lengths, at, at + 8 * n * L, at + 8 * n * L + 4 * n * C,
                               g.data_ptr()),) + (None,) * 8


def _want_candidates(logits, tokens, lengths):
    _want_floating(logits, "logits", 3, None, (torch.float32, torch.bfloat16, torch.float16))
    dev = logits.device
    _want(tokens, "tokens", torch.int32, 3, dev)
    _want(lengths, "lengths", torch.int32, 2, dev)
    n, L, V = logits.shape
    if tokens.shape[0] != n or tokens.shape[2] != L or lengths.shape != tokens.shape[:2]:
        raise ValueError("tokens must be [n, C, L] and lengths [n, C] with n, L matching logits [n, L, V]")
    if L == 0 or V == 0:
        raise ValueError("L and V must be positive")
    if tokens.shape[1] > 8192:
        raise ValueError("at most 8192 candidates per request")
    return dev


def sequence_logp(logits, tokens, lengths, stream=None):
    """Log-probabilities of candidate sequences under their request's logits
    (C ABI ft_sequence_logp_device), differentiable in the logits:

        logp[i, j] = sum of log_softmax(logits[i, l])[tokens[i, j, l]] over l < lengths[i, j]

    logits: float32, bfloat16 or float16 [n, L, V]; tokens int32 [n, C, L]
    (read as unsigned) and lengths int32 [n, C], as bs_tbs_device returns
    them: empty result slots have length 0 and score 0.  Returns float32
    [n, C], summed in 64 bits.  A length outside [0, L] gives NaN and no
    gradient.  A token id >= V, and any token of a position whose logits are
    all -inf, has log-probability -inf.  The gradient is deterministic; the
    backward pass runs on the forward call's stream."""
    dev = _want_candidates(logits, tokens, lengths)
    with _On(dev, stream, logits, tokens, lengths):
        if logits.requires_grad and torch.is_grad_enabled():
            return _SequenceLogp.apply(logits, tokens, lengths)
        return _scores(logits, tokens, lengths)[0]


def preference_loss(logits, tokens, lengths, ref_logp, chosen, rejected, beta=0.1, label_smoothing=0.0,
                    reduction="mean", stream=None):
    """Preference loss on pairs of candidate sequences (C ABI
    ft_preference_loss_device), differentiable in the logits:

        margin = beta * ((logp[c] - ref_logp[c]) - (logp[r] - ref_logp[r]))
        loss = (1 - label_smoothing) * softplus(-margin) + label_smoothing * softplus(margin)

    with logp = sequence_logp(logits, tokens, lengths), ref_logp float32
    [n, C] the scores under a reference (a constant), and chosen, rejected
    int32 [n, P] the pairs' candidate slots.  A pair with a negative slot is
    absent; one with a slot >= C makes the loss NaN.  reduction: "mean" over
    the pairs that are there (0 without any) or "sum".  Returns (loss, a
    float32 scalar, and margin, float32 [n, P], 0 for absent pairs, without
    gradient)."""
    dev = _want_candidates(logits, tokens, lengths)
    n, C = lengths.shape
    _want(ref_logp, "ref_logp", torch.float32, 2, dev)
    _want(chosen, "chosen", torch.int32, 2, dev)
    _want(rejected, "rejected", torch.int32, 2, dev)
    if ref_logp.shape != lengths.shape:
        raise ValueError("ref_logp must be [n, C]")
    if chosen.shape[0] != n or rejected.shape != chosen.shape:
        raise ValueError("chosen and rejected must both be [n, P]")
    if C == 0:
        raise ValueError("there are no candidates")
    if ref_logp.requires_grad and torch.is_grad_enabled():
        raise ValueError("ref_logp is a constant of the loss: detach it")
    beta, label_smoothing = float(beta), float(label_smoothing)
    if not math.isfinite(ctypes.c_float(beta).value):
        raise ValueError("beta must be finite in 32 bits")
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError("label_smoothing must be in [0, 1]")
    if reduction not in ("mean", "sum"):
        raise ValueError("reduction must be 'mean' or 'sum'")
    args = (logits, tokens, lengths, ref_logp, chosen, rejected, beta, label_smoothing, reduction == "mean")
    with _On(dev, stream, *args[:6]):
        if logits.requires_grad and torch.is_grad_enabled():
            return _PreferenceLoss.apply(*args)
        return _preference(*args)[:2]

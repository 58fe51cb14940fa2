"""What the serving operators refuse before any GPU work, and how their wrappers order streams
(on the CPU)."""
import ctypes

import numpy as np
import pytest


def _refused(llmrs, rc, words):
    assert rc == llmrs.EINVAL
    text = llmrs.lib().llmrs_last_error().decode()
    assert words in text, text


def _verify(llmrs, entry, ld=100, vocab=100, n=3, seqs=1, draft=4096, n_drafts=2, ldq=100):
    L = llmrs.lib()
    count = (n_drafts,) if entry == "llmrs_verify_draft_counted" else ()
    return getattr(L, entry)(None, 4096, ld, llmrs.F32, vocab, n, seqs, 4096, draft, 4096, ldq, *count, 4096, None, 4096,
                             4096, None, None, 0)


def test_counted_drafts_are_checked(llmrs):
    E = "llmrs_verify_draft_counted"
    _refused(llmrs, _verify(llmrs, E), "ctx is NULL")
    _refused(llmrs, _verify(llmrs, E, draft=None), "n_drafts 2")
    _refused(llmrs, _verify(llmrs, E, n_drafts=-1), "n_drafts -1")
    _refused(llmrs, _verify(llmrs, E, draft=None, n_drafts=0), "ctx is NULL")  # no drafts: rows behind the last sequence
    _refused(llmrs, _verify(llmrs, E, n=70000), "n_rows")
    _refused(llmrs, _verify(llmrs, E, ldq=99), "strides")
    _refused(llmrs, _verify(llmrs, "llmrs_verify_draft", draft=None), "no drafted tokens")
    _refused(llmrs, _verify(llmrs, "llmrs_verify_draft", draft=None, n=1), "ctx is NULL")


def test_vocabularies_past_32_bit_steps_are_refused(llmrs):
    n = ctypes.c_size_t(0)
    for vocab in ((1 << 30) + 1, (1 << 31) - 8192, (1 << 31) - 1):
        for entry in ("llmrs_verify_draft", "llmrs_verify_draft_counted"):
            _refused(llmrs, _verify(llmrs, entry, vocab=vocab, ld=1 << 31, ldq=1 << 31), "vocab")
        _refused(llmrs, llmrs.lib().llmrs_verify_draft_workspace(5, vocab, ctypes.byref(n)), "bad arguments")
    assert llmrs.lib().llmrs_verify_draft_workspace(5, 1 << 30, ctypes.byref(n)) == llmrs.OK
    assert n.value >= 5 * (1 << 30) // 8192 * 16


# ------------------------------------------------------------------ the Python wrappers
class _Gpu:
    """A context's number of its GPU, without the GPU."""
    h = None

    def __init__(self, device):
        self.device = device


class _Strange:
    """What a torch tensor on GPU 1 says of itself."""

    def __init__(self, shape, dtype):
        self.shape, self.dtype, self.nbytes = shape, dtype, 4096

    def get_device(self):
        return 1


def _tensor(llmrs, shape, dtype, device=0):
    t = object.__new__(llmrs.DeviceTensor)  # memory that no call gets to
    t.ctx, t.shape, t.dtype, t.ptr = _Gpu(device), shape, np.dtype(dtype), ctypes.c_void_p(4096)
    t.nbytes = int(np.prod(shape)) * t.dtype.itemsize
    return t


def _wrappers(llmrs, device=0):
    """name -> (call, its tensors) of each wrapper, on GPU `device`"""
    T = lambda *shape, dtype=np.float32: _tensor(llmrs, shape, dtype, device)  # noqa: E731
    I = lambda *shape: T(*shape, dtype=np.int32)  # noqa: E731
    ctx = _Gpu(device)
    be = llmrs.CudaBackend(ctx)
    codes = lambda: T(8, 2, 16, 64, dtype=np.int8)  # noqa: E731
    cache = llmrs.Kv8Cache(ctx, 8, 16, 2, 64, k_codes=codes(), v_codes=codes(), k_scales=T(8, 2), v_scales=T(8, 2))
    batch = llmrs.SeqBatch(I(3), I(2), I(2, 4))
    rope = dict(rope_cos=T(64, 32), rope_sin=T(64, 32))
    return {
        "append": (lambda **a: be.kv8_append(cache, batch, **a), dict(k=T(5, 128), v=T(5, 128), **rope)),
        "read": (lambda **a: be.kv8_read(cache, **a), dict(pages=I(3), k_out=T(3, 2, 16, 64), v_out=T(3, 2, 16, 64))),
        "attention": (lambda **a: be.kv8_attention(cache, batch, **a),
                      dict(q=T(5, 256), out=T(5, 256), workspace=T(64), **rope)),
        "verify": (be.verify_draft, dict(logits=T(5, 100), row_start=I(3), draft_tokens=I(3), draft_probs=T(3, 100),
                                         uniforms=T(5), tokens=I(5), accepted=I(2), token_probs=T(5), temperature=T(2),
                                         workspace=T(64))),
    }


def _all_right(llmrs, call, args):
    """The call gets as far as the C entry, which has no context."""
    with pytest.raises(llmrs.LlmrsError) as e:
        call(**args)
    assert "ctx is NULL" in str(e.value)


@pytest.mark.parametrize("op", ["append", "read", "attention", "verify"])
def test_tensors_of_the_host_and_of_other_gpus_are_refused(llmrs, op):
    import torch
    call, args = _wrappers(llmrs)[op]
    _all_right(llmrs, call, args)
    kinds = {np.dtype(np.float32): torch.float32, np.dtype(np.int32): torch.int32, np.dtype(np.int8): torch.int8}
    for name, x in args.items():
        for other in (torch.zeros(x.shape, dtype=kinds[x.dtype]), _Strange(x.shape, x.dtype),
                      _tensor(llmrs, x.shape, x.dtype, device=1)):
            with pytest.raises(ValueError, match="not on GPU 0|two arrays"):  # numpy's and torch's types differ
                call(**dict(args, **{name: other}))


def test_caches_and_batches_of_the_host_and_of_other_gpus_are_refused(llmrs):
    import torch
    for op, (call, args) in _wrappers(llmrs, device=1).items():
        _all_right(llmrs, call, args)
    I = lambda *shape, device=0: _tensor(llmrs, shape, np.int32, device)  # noqa: E731
    host = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    for arrays in ((host(3), host(2), host(2, 4)), (host(3), I(2), I(2, 4)), (I(3), host(2), I(2, 4)),
                   (I(3), I(2), host(2, 4)), (I(3), I(2), I(2, 4, device=1))):
        with pytest.raises(ValueError, match="host|GPU"):
            llmrs.SeqBatch(*arrays)
    pools = lambda device: dict(k_codes=_tensor(llmrs, (8, 2, 16, 64), np.int8, device),  # noqa: E731
                                v_codes=_tensor(llmrs, (8, 2, 16, 64), np.int8, device),
                                k_scales=_tensor(llmrs, (8, 2), np.float32, device),
                                v_scales=_tensor(llmrs, (8, 2), np.float32, device))
    with pytest.raises(ValueError, match="not on GPU 0"):
        llmrs.Kv8Cache(_Gpu(0), 8, 16, 2, 64, **dict(pools(0), v_codes=torch.zeros(8, 2, 16, 64, dtype=torch.int8)))
    there, here = llmrs.Kv8Cache(_Gpu(1), 8, 16, 2, 64, **pools(1)), llmrs.Kv8Cache(_Gpu(0), 8, 16, 2, 64, **pools(0))
    be, rows = llmrs.CudaBackend(_Gpu(0)), _tensor(llmrs, (5, 128), np.float32)
    with pytest.raises(ValueError, match="another GPU"):
        be.kv8_append(there, llmrs.SeqBatch(I(3), I(2), I(2, 4)), rows, rows)
    with pytest.raises(ValueError, match="another GPU"):
        be.kv8_attention(here, llmrs.SeqBatch(I(3, device=1), I(2, device=1), I(2, 4, device=1)), rows, rows)


def test_draft_probs_have_a_row_for_each_draft(llmrs):
    """None alone means certain drafts: an empty array beside drafted tokens is a wrong shape."""
    call, args = _wrappers(llmrs)["verify"]
    T = lambda n: _tensor(llmrs, (n, 100), np.float32)  # noqa: E731
    none = _tensor(llmrs, (0,), np.int32)
    for draft, probs in ((args["draft_tokens"], T(0)), (args["draft_tokens"], T(2)), (none, T(3)), (None, T(3))):
        with pytest.raises(ValueError, match="distributions"):
            call(**dict(args, draft_tokens=draft, draft_probs=probs))
    for draft, probs in ((args["draft_tokens"], None), (none, T(0)), (None, T(0)), (none, None), (None, None)):
        _all_right(llmrs, call, dict(args, draft_tokens=draft, draft_probs=probs))


# ------------------------------------------------------------------ streams
class _Entries:
    """Stands for the C library: notes the calls."""

    def __init__(self, fails):
        self.said, self.fails = [], fails

    def llmrs_ctx_wait_stream(self, h, s):
        self.said.append(("ctx behind", s))
        return 0

    def llmrs_stream_wait_ctx(self, h, s):
        self.said.append(("stream behind", s))
        return 0

    def llmrs_last_error(self):
        return b"as told"

    def entry(self, h, *args):
        self.said.append(("call", args))
        return 1 if self.fails else 0


@pytest.mark.parametrize("fails", [False, True])
@pytest.mark.parametrize("foreign", [False, True])
@pytest.mark.parametrize("own,torchs", [(None, 0), (0, 0), (7, 7), (0, 7), (7, 0)])
def test_calls_are_ordered_with_torch_s_stream(llmrs, monkeypatch, own, torchs, foreign, fails):
    L = _Entries(fails)
    monkeypatch.setattr(llmrs, "lib", lambda: L)
    monkeypatch.setattr(llmrs, "_raw_stream", lambda device: torchs)
    be = llmrs.CudaBackend(_Gpu(0))
    be.ctx.raw_stream = own
    if fails:
        with pytest.raises(llmrs.LlmrsError):
            be._launch(foreign, L.entry, 1, 2)
    else:
        be._launch(foreign, L.entry, 1, 2)
    call = [("call", (1, 2))]
    if foreign and own != torchs:  # torch's stream waits even behind a call that failed
        call = [("ctx behind", torchs)] + call + [("stream behind", torchs)]
    assert L.said == call


def test_stream_entries_are_checked(llmrs):
    _refused(llmrs, llmrs.lib().llmrs_ctx_wait_stream(None, None), "ctx is NULL")
    _refused(llmrs, llmrs.lib().llmrs_stream_wait_ctx(None, None), "ctx is NULL")

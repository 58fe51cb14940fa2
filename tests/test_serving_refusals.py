"""What the serving operators' entries refuse before any GPU work (on the CPU)."""
import ctypes


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

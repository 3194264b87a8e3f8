"""CPU checks of the log probabilities: what a call refuses, and how rows are cut into slices."""
import ctypes as C

import pytest

import aoship

P = 1 << 12  # any aligned address: nothing is read


def _check(logits=P, bf16=0, T=3, vocab=100, stride=100, targets=P, **kw):
    f = aoship.lib().aoship_internal_logprobs_check
    f.restype, f.argtypes = C.c_int, [C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int64, C.c_void_p, C.c_void_p]
    d = dict(logprob=P, rank=P, entropy=P, top_ids=P, top_logprobs=P, n_top=5)
    d.update(kw)
    return f(logits, bf16, T, vocab, stride, targets, C.byref(aoship._LogProbsOut(**d)))


def test_good_calls_pass():
    assert _check() == 0 and _check(bf16=1, logits=P + 2, stride=103) == 0
    assert _check(targets=None, logprob=None, rank=None) == 0
    assert _check(n_top=0, top_ids=None, top_logprobs=None) == 0
    assert _check(n_top=5, top_ids=None, top_logprobs=None) == 0  # (a number without outputs asks for nothing)
    assert _check(T=1 << 26, vocab=1 << 30, stride=1 << 30) == 0 and _check(vocab=32, stride=32, n_top=32) == 0


def test_no_rows_is_nothing_to_do():
    assert _check(T=0) == 1 and _check(T=0, logits=None) == 1
    assert _check(T=0, n_top=33) == -1  # (bad arguments are refused all the same)


@pytest.mark.parametrize("kw", [dict(T=-1), dict(T=(1 << 26) + 1), dict(vocab=0), dict(vocab=(1 << 30) + 1, stride=1 << 31),
                                dict(stride=99), dict(stride=-100), dict(stride=1 << 40), dict(logits=None),
                                dict(logits=P + 2), dict(logits=P + 1, bf16=1), dict(n_top=-1), dict(n_top=33),
                                dict(vocab=4, n_top=5), dict(n_top=0), dict(targets=None), dict(targets=P + 2),
                                dict(targets=None, logprob=None), dict(logprob=P + 1), dict(rank=P + 2),
                                dict(entropy=P + 3), dict(top_ids=P + 2), dict(top_logprobs=P + 1)],
                         ids=lambda k: "-".join(k))
def test_bad_calls_are_refused(kw):
    assert _check(**kw) == -1
    assert aoship.last_error().startswith("aoship_logprobs")


def test_null_handles():
    L = aoship.lib()
    assert L.aoship_logprobs(None, None, 0, 0, 0, 0, None, None) == -1 and "null handle" in aoship.last_error()
    assert L.aoship_logprobs_set_stream(None, None) == -1
    L.aoship_logprobs_free(None)
    assert L.aoship_model_score(None, None, 0, 0, None, None, None, None) == -1 and "null" in aoship.last_error()


@pytest.mark.parametrize("T", [1, 2, 3, 7, 64, 300, 1023, 1024, 1025, 2047, 2048, 2049, 1 << 26])
@pytest.mark.parametrize("vocab", [1, 31, 2047, 4095, 4096, 4097, 50257, 152064, 999983, 1 << 24, 1 << 30])
def test_slices_cover_a_row_within_the_workspace(T, vocab):
    f = aoship.lib().aoship_internal_logprobs_shape
    f.restype, f.argtypes = C.c_int, [C.c_int, C.c_int, C.POINTER(C.c_int)]
    span = C.c_int()
    n = f(T, vocab, C.byref(span))
    assert 1 <= n <= 1024 and n * span.value >= vocab and (n - 1) * span.value < vocab
    if n > 1:
        assert T * n <= 2048 and span.value % 32 == 0 and span.value >= 2048


@pytest.mark.parametrize("T", [1, 2, 3, 7, 100, 255, 256, 257, 341, 342, 511, 512, 513, 1023, 1024, 1025, 1 << 26])
@pytest.mark.parametrize("vocab", [4096, 50257, 152064, 524287, 1 << 20, (1 << 21) + 1, 1 << 24, 1 << 30])
def test_slices_stay_within_the_handles_workspace(T, vocab):
    """The workspace holds the pieces of 1024 workgroups and as many rows' counters, and a thread joins four slices of a row."""
    f = aoship.lib().aoship_internal_logprobs_shape
    f.restype, f.argtypes = C.c_int, [C.c_int, C.c_int, C.POINTER(C.c_int)]
    span = C.c_int()
    n = f(T, vocab, C.byref(span))
    assert 1 <= n <= 1024
    if n > 1:
        assert T * n <= 1024 and T <= 1024

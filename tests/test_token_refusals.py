"""What the token operators and gradient clipping refuse: every case below is
turned away before anything is launched, so it runs without a GPU."""
import ctypes

import pytest

ARG = -1  # TP_ERR_ARG
P = 4096  # an address no case gets as far as reading
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def lib():
    import os

    from tpcuda import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from tpcuda.build import build
        build()
    return _lib.load()


def refused(lib, status, word):
    assert status == ARG, (status, lib.tp_last_error())
    assert word in lib.tp_last_error().decode(), lib.tp_last_error()


LOGPROBS = dict(logits=P, ld=100, ids=P, kind=1, rows=4, vocab=100, topk=3, logp=P, entropy=P, stats=P, top_ids=P,
                top_logp=P)


@pytest.mark.parametrize("change, word", [
    (dict(rows=-1), "rows"), (dict(rows=2 ** 31), "rows"), (dict(vocab=0), "vocabulary"),
    (dict(vocab=2 ** 24 + 1, ld=2 ** 25), "vocabulary"), (dict(ld=99), "row stride"), (dict(topk=-1), "topk"),
    (dict(topk=33), "topk"), (dict(vocab=2, topk=3), "topk"), (dict(kind=2), "ids_kind"), (dict(kind=-1), "ids_kind"),
    (dict(logits=None), "logits"), (dict(ids=None), "token ids"), (dict(top_ids=None), "alternatives"),
    (dict(top_logp=None), "alternatives"), (dict(logits=P + 2), "aligned"), (dict(ids=P + 1), "aligned"),
    (dict(logp=P + 2), "aligned"), (dict(entropy=P + 2), "aligned"), (dict(stats=P + 2), "aligned"),
    (dict(top_ids=P + 2), "aligned"), (dict(top_logp=P + 3), "aligned")])
def test_logprobs(lib, change, word):
    refused(lib, lib.tpk_token_logprobs(*{**LOGPROBS, **change}.values()), word)


BACKWARD = dict(logits=P, ld=100, ids=P, kind=1, stats=P, entropy=P, dlogp=P, dentropy=P, rows=4, vocab=100,
                dlogits=2 * P, ldd=100)


@pytest.mark.parametrize("change, word", [
    (dict(rows=-1), "rows"), (dict(vocab=0), "vocabulary"), (dict(ld=99), "row stride"), (dict(ldd=99), "row stride"),
    (dict(kind=3), "ids_kind"), (dict(logits=None), "NULL"), (dict(stats=None), "NULL"), (dict(dlogits=None), "NULL"),
    (dict(ids=None), "token ids"), (dict(entropy=None), "entropy"), (dict(dlogits=P, ldd=101), "in place"),
    (dict(dlogits=P + 1), "aligned"), (dict(ids=P + 2), "aligned"), (dict(stats=P + 2), "aligned"),
    (dict(entropy=P + 2), "aligned"), (dict(dlogp=P + 1), "aligned"), (dict(dentropy=P + 2), "aligned")])
def test_logprobs_backward(lib, change, word):
    refused(lib, lib.tpk_token_logprobs_backward(*{**BACKWARD, **change}.values()), word)


EMBED = dict(table=P, ld=8, ids=P, kind=0, n=5, vocab=10, dim=8, scale=1.0, out=2 * P, ldo=8)


@pytest.mark.parametrize("change, word", [
    (dict(n=-1), "tokens"), (dict(n=2 ** 31 - 1), "tokens"), (dict(vocab=0), "vocabulary"),
    (dict(vocab=2 ** 24 + 1), "vocabulary"), (dict(dim=-1), "width"), (dict(dim=2 ** 31, ld=2 ** 31, ldo=2 ** 31), "width"),
    (dict(ld=7), "row stride"), (dict(ldo=7), "row stride"), (dict(kind=2), "ids_kind"), (dict(table=None), "NULL"),
    (dict(ids=None), "NULL"), (dict(out=None), "NULL"), (dict(out=P + 1), "aligned"), (dict(out=P), "input")])
def test_embedding(lib, change, word):
    refused(lib, lib.tpk_token_embedding(*{**EMBED, **change}.values()), word)


GRAD = dict(dout=P, ldo=8, ids=P, kind=0, n=5, vocab=10, dim=8, scale=1.0, pad=-1, accumulate=0, dtable=2 * P, ld=8, ws=P,
            ws_bytes=1 << 20)


@pytest.mark.parametrize("change, word", [
    (dict(n=-1), "tokens"), (dict(vocab=0), "vocabulary"), (dict(dim=-1), "width"), (dict(ld=7), "row stride"),
    (dict(ldo=7), "row stride"), (dict(kind=2), "ids_kind"), (dict(pad=-2), "padding_id"), (dict(pad=10), "padding_id"),
    (dict(accumulate=2), "accumulate"), (dict(dout=None), "NULL"), (dict(ids=None), "NULL"),
    (dict(dtable=None), "NULL"), (dict(ws_bytes=-1), "workspace"), (dict(n=5000, ws_bytes=8), "workspace"),
    (dict(n=5000, ws=None), "workspace"), (dict(ws=P + 4), "workspace"), (dict(dtable=P + 2), "aligned"),
    (dict(dtable=P), "input")])
def test_embedding_backward(lib, change, word):
    refused(lib, lib.tpk_token_embedding_backward(*{**GRAD, **change}.values()), word)


def test_embedding_workspace(lib):
    b = ctypes.c_int64(-1)
    assert lib.tpk_token_embedding_backward_ws(16384, 32000, 4096, ctypes.byref(b)) == 0 and b.value > 0
    assert lib.tpk_token_embedding_backward_ws(513, 10, 8, ctypes.byref(b)) == 0 and b.value > 0
    assert lib.tpk_token_embedding_backward_ws(512, 32000, 4096, ctypes.byref(b)) == 0 and b.value == 0
    refused(lib, lib.tpk_token_embedding_backward_ws(-1, 10, 8, ctypes.byref(b)), "tokens")
    refused(lib, lib.tpk_token_embedding_backward_ws(1, 0, 8, ctypes.byref(b)), "vocabulary")
    refused(lib, lib.tpk_token_embedding_backward_ws(1, 10, 8, None), "bytes")


@pytest.mark.parametrize("norm_type, max_norm, word", [
    (0.0, 1.0, "norm_type"), (3.0, 1.0, "norm_type"), (-INF, 1.0, "norm_type"), (NAN, 1.0, "norm_type"),
    (2.0, -1.0, "max_norm"), (2.0, NAN, "max_norm"), (INF, -INF, "max_norm")])
def test_clip(lib, norm_type, max_norm, word):
    ids = (ctypes.c_int64 * 1)(1)
    refused(lib, lib.tp_clip_grad_norm_multi(ids, 1, norm_type, max_norm, None), word)
    refused(lib, lib.tpk_group_clip_grad_norm(1, norm_type, max_norm, P), word)
    refused(lib, lib.tpk_group_grad_norm(1, norm_type, max_norm, P), word)


def test_clip_groups_and_counts(lib):
    one = (ctypes.c_int64 * 1)(987654321)
    refused(lib, lib.tpk_group_clip_grad_norm(987654321, 2.0, 1.0, P), "unknown tensor group")
    refused(lib, lib.tpk_group_grad_norm(987654321, 2.0, 1.0, P), "unknown tensor group")
    refused(lib, lib.tpk_group_grad_norm(1, 2.0, 1.0, None), "NULL")
    refused(lib, lib.tpk_adam_group_scaled(987654321, 0, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1e-3, 1.0, P), "unknown tensor group")
    refused(lib, lib.tpk_adam_group_scaled(1, 2, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1e-3, 1.0, P), "kind")
    refused(lib, lib.tpk_adam_group_scaled(1, 0, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1e-3, 1.0, None), "NULL")
    refused(lib, lib.tp_clip_grad_norm_multi(one, -1, 2.0, 1.0, None), "negative")
    refused(lib, lib.tp_clip_grad_norm_multi(one, 1, 2.0, 1.0, None), "Unknown tensor id")
    refused(lib, lib.tp_adam_clip_step_multi(2, one, one, one, one, 1, *[0.1] * 8, None), "kind")
    refused(lib, lib.tp_adam_clip_step_multi(0, one, one, one, one, -1, *[0.1] * 8, None), "negative")
    refused(lib, lib.tp_adam_clip_step_multi(0, one, one, one, one, 1, *[0.1] * 7, -1.0, None), "max_norm")


def test_handles_that_name_no_tensor(lib):
    bad = 987654321
    for status in (lib.tp_token_logprobs(bad, bad, 0, None, None, None, None, None),
                   lib.tp_token_logprobs_backward(bad, 0, bad, bad, bad, bad, None),
                   lib.tp_token_embedding(bad, bad, 1.0, None),
                   lib.tp_token_embedding_backward(bad, bad, 10, 1.0, -1, 0, None)):
        refused(lib, status, "Unknown tensor id")


def test_empty_calls_do_nothing(lib):
    assert lib.tpk_token_logprobs(None, 100, None, 0, 0, 100, 0, None, None, None, None, None) == 0
    assert lib.tpk_token_logprobs_backward(None, 100, None, 0, None, None, None, None, 0, 100, None, 100) == 0
    assert lib.tpk_token_embedding(None, 8, None, 0, 0, 10, 8, 1.0, None, 8) == 0
    assert lib.tpk_token_embedding(None, 0, None, 0, 5, 10, 0, 1.0, None, 0) == 0
    assert lib.tpk_token_embedding_backward(None, 0, None, 0, 5, 10, 0, 1.0, -1, 0, None, 0, None, 0) == 0

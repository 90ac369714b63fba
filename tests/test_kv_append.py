"""frq_kv_append_dev without a GPU: every refusal that needs none (checked
before the context, so a null context shows it was reached)."""
import ctypes as C

import pytest

import fieldrun_amd as fa
from test_kv import A, BAD_CACHES, desc, message


def append(d=None, how=None, x=A, pitch=512, n_head=4, pos=A, slot=A, n=3, q=A, q_pitch=256, **change):
    f = dict(bias=None, q_norm=None, k_norm=None, eps=1e-6, freq=A, rot=64, pairs=0)
    f.update(change)
    d = C.byref(desc()) if d is None else d
    return fa.lib.frq_kv_append_dev(None, d, C.byref(fa._Rotary(*f.values())) if how is None else how, x, pitch, n_head,
                                    pos, slot, n, q, q_pitch)


@pytest.mark.parametrize("change,code,word", BAD_CACHES)
def test_bad_descriptors_are_refused(change, code, word):
    assert append(C.byref(desc(**change)), pitch=1 << 20, q_pitch=1 << 20) == code and word in message(), message()


@pytest.mark.parametrize("change,word", [
    (dict(rot=12), "rot"), (dict(rot=72), "rot"), (dict(rot=1 << 63), "rot"), (dict(pairs=2), "pairs"),
    (dict(pairs=-1), "pairs"), (dict(eps=-1e-9), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
    (dict(n_head=0), "n_head"), (dict(n_head=3), "n_head"), (dict(n_head=1 << 40), "n_head"), (dict(pitch=511), "pitch"),
    (dict(q_pitch=255), "pitch"), (dict(pitch=1 << 41), "pitch"), (dict(q_pitch=1 << 41), "pitch"),
    (dict(n=1 << 32), "too many"), (dict(n=1 << 31), "too many"), (dict(n=1 << 29), "too many"),
    (dict(n=1 << 63), "too many"), (dict(x=None), "null pointer"), (dict(q=None), "null pointer"),
    (dict(slot=None), "null pointer"), (dict(pos=None), "null pointer"), (dict(freq=None), "null pointer"),
    ({}, "null context"), (dict(rot=0, pos=None, freq=None), "null context"),
    (dict(n=0, x=None, q=None, slot=None, pos=None, freq=None), "null context"),
])
def test_bad_calls_are_refused(change, word):
    assert append(**change) == fa.FRQ_ERR_ARG and word in message(), message()


def test_null_rotary():
    d = C.byref(desc())
    assert fa.lib.frq_kv_append_dev(None, d, None, A, 512, 4, A, A, 1, A, 256) == fa.FRQ_ERR_ARG
    assert "null rotary" in message()


def test_rows_that_no_launch_holds_are_refused():
    """A grid has fewer than 2^32 threads: a workgroup for every two rows, one for
    every 32 of each of 2 kv heads."""
    most = (2 ** 24 - 1) * 16 // 9
    for n in (most + 32, 1 << 25, 1 << 26):
        assert append(n=n) == fa.FRQ_ERR_ARG and "too many" in message(), message()
    for n in (most - 32, 1 << 24):
        assert append(n=n) == fa.FRQ_ERR_ARG and "null context" in message(), message()

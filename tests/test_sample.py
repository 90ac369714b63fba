"""frq_sample_dev without a GPU: its refusals and its workspace's size."""
import pytest

import fieldrun_amd as fa
from test_kv import A, message


def sample(x=A, pitch=1000, m=3, n=1000, temp=A, topk=A, topp=A, minp=A, u=A, token=A, prob=A, ws=A, ws_bytes=1 << 40):
    return fa.lib.frq_sample_dev(None, x, pitch, m, n, temp, topk, topp, minp, u, token, prob, ws, ws_bytes)


@pytest.mark.parametrize("change,word", [
    (dict(n=0), "n must"), (dict(n=(1 << 24) + 1, pitch=1 << 30), "n must"), (dict(m=(1 << 20) + 1), "too many"),
    (dict(m=1 << 63), "too many"), (dict(pitch=999), "pitch"), (dict(pitch=1 << 41), "pitch"), (dict(x=None), "null pointer"),
    (dict(u=None), "null pointer"), (dict(token=None), "null pointer"), (dict(ws=A + 8), "16-byte"), ({}, "null context"),
    (dict(temp=None, topk=None, topp=None, minp=None, prob=None), "null context"),
    (dict(m=0, x=None, u=None, token=None), "null context"),
])
def test_bad_calls_are_refused(change, word):
    assert sample(**change) == fa.FRQ_ERR_ARG and word in message(), message()


def test_workspace():
    size = fa.lib.frq_sample_ws
    assert size(0, 5) == size(5, 0) == size(1, (1 << 24) + 1) == size((1 << 20) + 1, 5) == 0
    for m in (1, 7, 64, 1000, 1 << 20):
        for n in (1, 3, 5000, 152064, 1 << 24):
            assert 0 < size(m, n) < m * (140000 + (n // 16384 + 41) * 7000)

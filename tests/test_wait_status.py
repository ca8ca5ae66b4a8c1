"""How a weight gradient that gave up a wait is reported, on the host.  No GPU: the word that a kernel would set
is set here."""

from __future__ import annotations

import threading
import time

import pytest
import torch

from adamw4bit_b200 import ZEEDENAdamW4Bit
from adamw4bit_b200 import _native as N
from adamw4bit_b200 import activations as A


@pytest.fixture
def words(monkeypatch):
    monkeypatch.setattr(N, "_wait_words", {})
    monkeypatch.setattr(N, "_new_wait_word", lambda: torch.zeros(1, dtype=torch.int32))
    return N._wait_words


def test_a_word_for_each_device(words):
    a, b = N.wait_status(0), N.wait_status(1)
    assert a != b and N.wait_status(0) == a
    words[1][0] = 1                                       # device 1's kernel
    assert N.wait_status(0) == a
    with pytest.raises(N.NativeError, match="cuda:1"):
        N.wait_status(1)
    assert N.wait_status(1) == b                          # said once


def test_the_check_raises_once_and_for_its_device(words):
    A.check_weight_grads(0, synchronize=False)            # nothing ran
    N.wait_status(0)
    N.wait_status(3)
    A.check_weight_grads(0, synchronize=False)
    words[0][0] = 1
    A.check_weight_grads(torch.device("cuda:3"), synchronize=False)
    A.check_weight_grads("cuda:3", synchronize=False)
    with pytest.raises(N.NativeError, match="not complete"):
        A.check_weight_grads(torch.device("cuda:0"), synchronize=False)
    A.check_weight_grads(0, synchronize=False)


def test_an_optimizer_does_not_step_with_it(words):
    p = torch.nn.Parameter(torch.zeros(128))
    opt = ZEEDENAdamW4Bit([p])
    opt.step()                                            # no gradient: nothing to launch
    N.wait_status(2)
    words[2][0] = 1
    with pytest.raises(N.NativeError, match="cuda:2"):
        opt.step()
    opt.step()

    def closure():
        words[2][0] = 1
        return torch.zeros(())

    with pytest.raises(N.NativeError):
        opt.step(closure)


def test_threads_share_the_first_word(words, monkeypatch):
    made = []

    def slow():
        time.sleep(0.05)
        made.append(torch.zeros(1, dtype=torch.int32))
        return made[-1]

    monkeypatch.setattr(N, "_new_wait_word", slow)
    got, gate = [], threading.Barrier(8)

    def first():
        gate.wait()
        got.append(N.wait_status(0))

    threads = [threading.Thread(target=first) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(set(got)) == 1 and len(made) == 1 and got[0] == made[0].data_ptr()

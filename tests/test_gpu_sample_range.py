"""Sampling from vocabularies of 2^20 logits and more, whose mass in units of 2^-44 of the
largest weight may pass 64 bits.

Equal logits are exact in whole units and in numpy's 64 bits: every token is the
definition's.  With other values a weight is off by half a unit at most, 2^-43 of the
largest at 2^21 logits: all of them together by 2^-22 where all err alike, and
2^10.5 2^-43 0.3 = 5e-11 as independent roundings, in masses of thousands here of which a
token is 1e-3 and more of the largest weight.  Random numbers come nearer than that to a
border once in some thousand rows at the very worst."""

import numpy as np
import pytest

import test_gpu_sample as ts

pytestmark = pytest.mark.gpu
SIZES = [(1 << 20) - 1, 1 << 20, 1500000, 1 << 21, (1 << 21) + 7]


@pytest.mark.parametrize("vocab", SIZES)
def test_equal_logits(vocab):
    ts.say("sample, equal logits", vocab)
    u = np.array([0.0, 0.1, 0.5, 0.75, 0.999], np.float32)
    x = np.full((u.size, vocab), 1.5, np.float32)
    for how in ({}, {"p": 0.25}, {"p": 0.75}, {"k": vocab // 2}, {"k": vocab - 1, "p": 0.5}, {"m": 0.5}, {"m": 1.0, "p": 0.75}, {"t": 0.0}):
        ts.agree(x, u, **how)


@pytest.mark.parametrize("vocab", SIZES)
def test_two_values(vocab):
    """Most of the row at the maximum, the rest at an eighth of its weight."""
    ts.say("sample, two values", vocab)
    rng = np.random.default_rng(vocab)
    u = (rng.integers(0, 1 << 12, 3) + 0.5) / (1 << 12)
    x = np.where(rng.random((3, vocab)) < 0.9, 3.0, 0.0).astype(np.float32)
    most = int((x[0] > 0).sum())
    for how in ({}, {"k": most + 5}, {"k": vocab - 9, "p": 0.25}, {"p": 0.5}, {"m": 0.5}):
        ts.agree(x, u, t=1.4, **how)


@pytest.mark.parametrize("sigma,likely", [(0.3, 0.0), (2.0, 10.0)])
def test_ordinary_rows(sigma, likely):
    ts.say("sample, many ordinary logits", sigma, likely)
    vocab = (1 << 21) + 7
    rng = np.random.default_rng(int(10 * sigma))
    x, u = ts.logits(rng, 2, vocab, sigma, likely, bf16=False), rng.random(2)
    for how in ({}, {"p": 0.9}, {"k": 300000}, {"k": 300000, "p": 0.8}, {"m": 0.01}, {"k": 40}):
        ts.agree(x, u, **how)


def test_sixteen_million_equal_logits():
    ts.say("sample, 2^24 equal logits")
    x = np.zeros((2, 1 << 24), np.float32)
    for how in ({}, {"p": 0.5}, {"k": 1 << 23, "p": 0.5}):
        ts.agree(x, [0.25, 0.8], **how)

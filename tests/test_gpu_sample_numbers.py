"""Random numbers of 64 bits just below 1, as numpy's generators give them, draw the last
kept token and are not refused."""

import numpy as np
import pytest

import test_gpu_sample as ts
from tvara_amd import _capi, native
from tvara_amd import gguf_writer as gf
from tvara_amd.sampling import sample_batch

pytestmark = pytest.mark.gpu
CLOSE = [1 - 2.0 ** -24, 1 - 2.0 ** -26, 1 - 2.0 ** -53]


def test_rows_of_logits():
    ts.say("sample, numbers near 1")
    x = np.zeros((3, 5000), np.float32)
    for how in ({}, {"top_p": 0.5}, {"top_k": 100}):
        got, _ = sample_batch(x, np.array(CLOSE), **how)
        assert got.tolist() == [{(): 4999, ("top_p",): 2499, ("top_k",): 99}[tuple(how)]] * 3
    for u in (1.0, 1 + 2.0 ** -40):
        with pytest.raises(_capi.InvalidArgument, match="parameters"):
            sample_batch(x[:1], np.array([u]))


def test_a_models_step(tmp_path):
    ts.say("sample sequences, numbers near 1")
    spec = gf.LlamaSpec()
    model = native.NativeModel(spec.write(tmp_path / "m.gguf"), max_blocks=16, block_tokens=4)
    a, b = model.new_sequence(), model.new_sequence()
    last = float(np.nextafter(np.float32(1), np.float32(0)))
    for u in CLOSE:
        assert model.sample_sequences([a], [3], np.array([u]))[0] == model.sample_sequences([b], [3], [last])[0]
    with pytest.raises(Exception, match="parameters"):
        model.sample_sequences([a], [3], [1.0])

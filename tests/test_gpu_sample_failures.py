"""A sampled step that fails half-way leaves nothing to the next one."""

import numpy as np
import pytest

import test_gpu_sample_sequences as tss
from tvara_amd import gguf_writer as gf
from tvara_amd import native

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [{"temperature": [-1.0, 1.0]}, {"top_p": [1.5, 1.0]}, {"min_p": [np.nan, 0.0]}])
def test_a_report_of_a_step_that_failed_is_not_the_next_ones(tmp_path, bad):
    """Widths without batched products: the first row is drawn before the second finds no block."""
    tss.say("sample sequences, reports", bad)
    spec = gf.LlamaSpec(matrix_type=gf.T_F32, hidden=40, intermediate=72, heads=4, kv_heads=2, vocab=90)
    path = spec.write(tmp_path / "m.gguf")
    model, twin = (native.NativeModel(path, max_blocks=3, block_tokens=4) for _ in range(2))
    a, b = model.new_sequence(), model.new_sequence()
    text = [3, 1, 4, 1]
    model.decode_batch(a, text)
    model.decode_batch(b, text[::-1])
    other = twin.new_sequence()
    twin.decode_batch(other, text)
    u = np.array([0.3, 0.6], np.float32)
    for _ in range(2):
        with pytest.raises(Exception) as failed:  # two full blocks of three
            model.sample_sequences([a, b], [5, 9], u, **bad)
        assert "sampling" not in str(failed.value)
    got, chances = model.sample_sequences([a], [5], u[:1], temperature=0.9)
    tss.expect(twin.decode_sequences([other], [5]), u[:1], got, chances, t=0.9)
    token = got[0]
    got, chances = model.sample_sequences([a], [token], u[1:])
    tss.expect(twin.decode_sequences([other], [token]), u[1:], got, chances)

"""Calls of the serving operators at their borders: the decoder's log probabilities without a step, many rows at once, status
words, queries of the device that fail."""
import numpy as np
import pytest

import serving_reference as ref
from serving_reference import Case, f64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available(), "a CUDA device is required"
    t.cuda.set_device(0)
    return t


def test_decoder_logprobs_need_a_step(torch, mvb, tmp_path):
    """Refused where the logits are of no step, of another head's, or of the step before a prompt."""
    path = str(tmp_path / "tiny.qwb")
    mvb.qwb.write_synthetic_qwb(path, mvb.qwb.QWEN_TINY, seed=11)
    dec = mvb.QwenDecoder(path, ctx=64)

    def refused():
        with pytest.raises(mvb.MatvecError, match="no step"):
            dec.logprobs([0], top=1)

    def fine(logits=None):
        logp, ent, top, top_logp = dec.logprobs([0], top=1)
        assert np.isfinite(logp[0]) and np.isfinite(ent) and logp[0] <= top_logp[0] <= 0
        assert logits is None or top[0] == int(np.argmax(logits))

    try:
        refused()
        fine(dec.forward(5, 0)[1])
        dec.full_head(False)  # the head in use already
        fine()
        dec.full_head(True)
        refused()
        fine(dec.forward(5, 0)[1])
        dec.full_head(False)
        refused()
        for feed in (dec.prefill, dec.prefill_tokenwise):
            fine(dec.forward(5, 0)[1])
            feed([3, 4, 5])
            refused()
            dec.decode(0)
            refused()
            dec.decode(2)
            fine()
        dec.prefill([3])
        refused()
        dec.trace(3, 0)
        fine()
    finally:
        dec.close()

"""Batch-1 decode with a vocabulary smaller than the LM head's grid (one partial maximum a CTA)."""
import numpy as np
import pytest

from oracle.oracle import OwnModel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [40, 500])
def test_small_vocabulary_decode(jd, orc, gpu_ctx, vocab):
    over = dict(vocab_size=vocab, seq_len=96)
    om = OwnModel(orc, orc.config(4, **over), 3, 0.05, False)
    eng = jd.Engine.own(gpu_ctx, jd.Model.seeded(jd.config_from_depth(4, **over), 3, 0.05, False), 1)
    try:
        prompt = np.random.default_rng(1).integers(0, vocab, 30)
        want, lg = [], None
        for i, t in enumerate(prompt):
            lg = om.forward(int(t), i)
        for i in range(8):
            want.append(int(np.argmax(lg)))
            lg = om.forward(want[-1], 30 + i)
        eng.set_prompt(prompt[None], [30])
        eng.run(1, 30 - 1 + 8)
        assert eng.history(1, 8)[0].tolist() == want
    finally:
        eng.close()
        om.close()

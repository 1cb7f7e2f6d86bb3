"""Steps of a beam search whose sums leave their range: the search says so, as generate does."""
import numpy as np
import pytest

import q35
from q35 import _lib as L

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("beams", [2, 6])
@pytest.mark.parametrize("mode", ["graph", "stream"])
def test_a_step_out_of_range_raises(beams, mode):
    """The id that the search chooses first has an embedding whose squares' sum passes 2^31 (512 values of about 10^5 and more): the
    prompt is in range, the step that takes that id is not."""
    d = q35.make_dims(hidden=512, ffn=1536, vocab=8192, n_layers=4, lin_heads=4, attn_heads=4, kv_heads=2)
    m = q35.TextForCausalLM(d, seed=3, tmax=40)
    prompt = np.arange(100, 109, dtype=np.int32)
    first, _ = q35.BatchDecoder(m, 1, 20).generate([prompt], 0, prefill=True)
    first = int(first[0, 0])
    assert first not in prompt
    scale = m.tensor("embed_tokens.scale", np.float32).reshape(d.vocab, -1)
    scale[first] *= np.float32(1e7)
    m.close()
    m = q35.TextForCausalLM(d, seed=3, tmax=40)
    m.set_tensor("embed_tokens.scale", scale)
    bt = q35.BatchDecoder(m, beams, 20)
    ids = bt.beam_search([prompt], beams, 1, mode=mode)  # (no step yet)
    assert ids[0][0][0].tolist() == [first]
    with pytest.raises(q35.Q35Error) as e:
        bt.beam_search([prompt], beams, 3, mode=mode)
    assert e.value.code == L.Q35_E_RANGE
    # generate in the same situation, and a check of steps made by hand
    with pytest.raises(q35.Q35Error) as e:
        bt.reset()
        bt.generate([prompt] * beams, 1, mode=mode, prefill=True)
    assert e.value.code == L.Q35_E_RANGE
    bt.reset()
    bt.generate([prompt] * beams, 0, mode=mode, prefill=True)
    bt.check()
    bt.step(mode=mode)
    with pytest.raises(q35.Q35Error) as e:
        bt.check()
    assert e.value.code == L.Q35_E_RANGE
    bt.check()  # (told once)
    bt.close()
    m.close()

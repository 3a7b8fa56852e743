"""An embedding with other rows than the vocabulary is no head."""
import numpy as np
import pytest
import torch

import model_gen as mg
from ditch_amd import abi, hipmem, synth
from ditch_amd.hip import DeviceError, Model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [49, 64])
def test_an_embedding_of_other_rows_than_the_vocabulary(dev, rows):
    spec = mg.dense(hidden=64, inter=64, layers=1, heads=2, kv_heads=1, head_dim=32, vocab=50, seed=3, tie=rows > 50)
    embed = torch.randn(rows, 64, generator=torch.Generator().manual_seed(1)) * 0.05
    spec.set("EMBED", synth.QUANTIZERS["bf16"](embed))
    model = Model(dev, spec)
    try:
        tokens, at = np.arange(5, dtype=np.uint32), [(0, p) for p in range(5)]
        if rows > 50:  # tied
            with pytest.raises(DeviceError, match="vocabulary"):
                model.head()
            with pytest.raises(DeviceError, match="vocabulary") as e:
                model.forward(tokens, at, logit_rows=[4])
            assert e.value.status == abi.INVALID_ARGUMENT
        else:  # the head is its own
            assert model.head().rows == 50
            assert np.isfinite(model.forward(tokens, at, logit_rows=[4])[1]).all()
        # hidden rows need no head
        bt, br = hipmem.Buffer.from_array(tokens), hipmem.Buffer.from_array(np.array(at, np.uint32))
        bw, out = hipmem.Buffer.from_array(np.array([4], np.uint64)), hipmem.Buffer(64 * 4)
        model.forward_hidden_device(bt.ptr, br.ptr, 5, 1, 5, bw.ptr, 1, out.ptr)
        dev.sync()
        assert np.isfinite(out.download(np.float32, (64,))).all()
    finally:
        model.free()

"""The models of test_gpt_rules_gpu.py at a length that the tensor-core attention kernels take: the gradients of the bias tables and of the projections are
small differences of large sums there, and are held to the same bar."""
import numpy as np
import pytest

from gradcraft_b200 import synth
from tests import test_gpt_rules_gpu as G
from tests.helpers import assert_grads_close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("arch", ["lngelu", "rmsswiglu"])
@pytest.mark.parametrize("opt", [dict(rel_buckets=7, rel_reach=33), dict(window=300, sinks=3, rel_buckets=32, rel_reach=128, dropout=0.1, dropout_seed=3)], ids=["bias", "all"])
def test_training_step(monkeypatch, arch, opt):
    for name, size in dict(V=96, T=600, C=128, H=2, L=2, F=256 if arch == "lngelu" else 384, B=2).items():
        monkeypatch.setattr(G, name, size)
    tr, w = G.make(arch, opt)
    ref = G.Reference(arch, w, opt, opt.get("dropout", 0.0))
    batches = [tuple(np.ascontiguousarray(x) for x in b) for b in synth.token_batches(3, 1, G.B, G.T, G.V)]
    tr.zero_grad()
    loss = sum(tr.forward_backward(x, y) for x, y in batches)
    want, grads = ref.loss_and_grads(batches)
    assert abs(loss - want) < 1e-5 * want
    assert_grads_close({k: v.reshape(grads[k].shape) for k, v in tr.get("grad").items()}, grads)
    tr.close()

"""The Decoder's bookkeeping of a shared prefix, on the host (no GPU: its buffers on the CPU, the integers that a launch would
carry written there): which cache rows a step reads and writes, and what is refused before anything runs."""
import numpy as np
import pytest
import torch
from ferrite_amd import lib, llama as G, ops
from oracle import llama as OL

needs_lib = pytest.mark.skipif(not lib.PATH.exists(), reason="libferrite_hip.so not built")
pytestmark = needs_lib


@pytest.fixture
def decoder(monkeypatch):
  """A Decoder without weights: 3 rows, 4 slots of 100 places."""
  monkeypatch.setattr(ops, "put_i32", lambda values, out: out.copy_(torch.from_numpy(np.ascontiguousarray(values, np.int32)).view(out.shape)))
  c = OL.smollm(layers=1, vocab=256, places=400)
  gc = G.model(**{k: getattr(c, k) for k in ("dim", "heads", "kv", "layers", "eps", "theta", "vocab", "ffn", "places", "rope", "tied")})
  d = G.Decoder.__new__(G.Decoder)
  d.c, d.mode, d.batch, d.context, d.device = gc, "bfp8", 3, 100, torch.device("cpu")
  d.hd = G.head(gc)
  d._buffers("bf16", 3, 100, 4)
  return d


def test_the_callers_counts_are_copied(decoder):
  # the caller's array changes after share_prefix: the rows are still placed by what the GPU reads with
  rows = np.array([70, 35, 0], np.int32)
  decoder.share_prefix(3, 70, rows=rows)
  rows[:] = 1
  decoder.set_rows([70, 40, 9], [0, 1, 2])
  assert decoder.shared.tolist() == [70, 35, 0] and decoder.rows.tolist() == [0, 100 + 5, 200 + 9]
  with pytest.raises(ValueError): decoder.set_rows([70, 20, 9], [0, 1, 2])  # (place 20 is the prefix's)

"""The Decoder's steps over a cache in pages, on the host (no GPU: its buffers on the CPU, the integers that a launch would carry written
there): what a step is given, and what is refused before anything runs; and a put whose q would lie over rows not yet read."""
import numpy as np
import pytest
import torch
from ferrite_amd import lib, llama as G, ops
from oracle import llama as OL
from test_paged_refusals import append

needs_lib = pytest.mark.skipif(not lib.PATH.exists(), reason="libferrite_hip.so not built")
pytestmark = needs_lib


@pytest.fixture
def decoder(monkeypatch):
  """A Decoder of two blocks without weights: 4 slots of 96 places, 24 pages of 16."""
  monkeypatch.setattr(ops, "put_i32", lambda values, out: out.copy_(torch.from_numpy(np.ascontiguousarray(values, np.int32)).view(out.shape)))
  c = OL.smollm(layers=2, vocab=256, places=400)
  gc = G.model(**{k: getattr(c, k) for k in ("dim", "heads", "kv", "layers", "eps", "theta", "vocab", "ffn", "places", "rope", "tied")})
  d = G.Decoder.__new__(G.Decoder)
  d.c, d.mode, d.batch, d.context, d.device = gc, "bfp8", 3, 96, torch.device("cpu")
  d.hd = G.head(gc)
  d.qkv_cols = (gc.heads + 2 * gc.kv) * d.hd
  d._buffers("bf16", 3, 96, 4)
  return d


def adapters(n, K, parts, rank=8):
  return ops.Adapters(torch.zeros(n, rank * len(parts), K), torch.zeros(n, sum(parts), rank), None, parts)


@pytest.mark.parametrize("kw", [dict(), dict(xd=lib.BF16, qd=lib.F32), dict(qd=lib.BF16), dict(rows=1, qd=lib.BF16), dict(rows=1, xd=lib.BF16),
                                dict(rows=1, xd=lib.BF16, qd=lib.F32, ldq=768)])
def test_q_over_rows_of_another_type_is_refused(kw):
  # (a wave's q would land on columns that another wave has not read, one row's too)
  lib.load()
  with pytest.raises(ValueError, match="qkv's own columns"): append(**kw)


def test_a_step_keeps_the_adapters_it_was_made_with(decoder):
  # the caller's list and dicts change after the step was made: what it reads stays, and stays alive
  parts = (576, 192, 192)
  ads = [dict(qkv=adapters(2, 576, parts)), dict(qkv=adapters(2, 576, parts))]
  first = ads[0]["qkv"]
  step = decoder.page_step(2, 2, 16, ads)
  ads[0]["qkv"], ads[1]["gate_up"] = adapters(2, 576, parts, 16), adapters(2, 576, (1536, 1536))
  ads.append({})
  assert len(step.adapters) == 2 and step.adapters[0]["qkv"] is first and "gate_up" not in step.adapters[1]


def test_an_adapter_that_is_not_there_is_refused(decoder):
  # (the kernel takes an id past the adapters for none: a request would be answered by the base model, or in some blocks alone)
  parts = (576, 192, 192)
  ads = [dict(qkv=adapters(3, 576, parts)), dict(o=adapters(3, 576, (576,)), down=adapters(3, 1536, (576,), 16))]
  ok = dict(tokens=[[1, 2], [3]], places=[0, 5], tables=[[0], [1]], page=16)
  step = decoder.page_step(2, 2, 16, ads)
  for of in ([0, 3], [-2, 0], [1 << 40, 0], [0], [0, 1, 2]):
    with pytest.raises(ValueError, match="adapter"): decoder.step_pages(**ok, adapters=ads, of=of)
    with pytest.raises(ValueError, match="adapter"): step.set([1, 2], [0, 5], [[0], [1]], of)
  for none in (None, [], [{}, {}]):
    with pytest.raises(ValueError, match="there are none"): decoder.step_pages(**ok, adapters=none, of=[-1, 0])
  with pytest.raises(ValueError, match="there are none"): decoder.page_step(2, 2, 16).set([1, 2], [0, 5], [[0], [1]], [0, -1])
  for other in (dict(o=adapters(2, 576, (576,))), dict(o=adapters(3, 576, (576,)), down=adapters(4, 1536, (576,)))):
    with pytest.raises(ValueError, match="as many adapters"): decoder.step_pages(**ok, adapters=[ads[0], other], of=[0, 1])
    with pytest.raises(ValueError, match="as many adapters"): decoder.page_step(2, 2, 16, [ads[0], other])
  step.set([7, 8], [0, 20], [[4], [1, 2]], [2, -1])
  assert step.ids.tolist() == [7, 8] and step.p0.tolist() == [0, 20] and step.of.tolist() == [2, -1] and step.tables.tolist() == [[4, -1], [1, 2]]
  step.set([7, 8], [0, 20], [[4], [1, 2]])
  assert step.of.tolist() == [-1, -1]
  plain = decoder.page_step(2, 2, 16)
  plain.set([7, 8], [0, 20], [[4], [1, 2]], [-1, -1])
  assert plain.of.tolist() == [-1, -1]

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


def test_a_slot_is_read_behind_the_places_it_was_filled_behind(decoder, monkeypatch):
  # prefill_batch fills slots behind the whole prefix by default: a row that shares less of it would read them from another row
  def launched(T): raise RuntimeError("the checks passed")
  monkeypatch.setattr(decoder, "_prefill_buffers", launched)
  def fill(*a, **kw):  # prefill_batch up to where it would launch
    with pytest.raises(RuntimeError, match="the checks passed"): decoder.prefill_batch(*a, **kw)
  decoder.share_prefix(3, 70, rows=[70, 35, 0])
  fill([[1, 2], [3, 4], [5, 6]])
  with pytest.raises(ValueError, match="slot 1 holds what follows 70 places of a prefix, not 35"): decoder.set_rows([72, 40, 2], [0, 1, 2])
  for where in (torch.tensor, list):
    with pytest.raises(ValueError, match="not 35"): decoder.set_rows(where([72, 37, 0]), where([0, 1, 2]))
  decoder.set_rows([72, 35, 0], [0, 1, 2])           # (a row that begins its slot anew reads nothing of it)
  fill([[1, 2], [3, 4], [5, 6]], shared=[70, 35, 0])
  decoder.set_rows([72, 37, 2], [0, 1, 2])
  with pytest.raises(ValueError, match="slot 1"): decoder.prefill_batch([[7]], slots=[1], p0=[72])          # (a second turn by the default)
  fill([[7]], slots=[1], p0=[37], shared=[35])
  with pytest.raises(ValueError, match="slot 0"): decoder.share_prefix(0, 20)               # (no whole prompt)
  decoder.share_prefix()
  with pytest.raises(ValueError, match="slot 0"): decoder.set_rows([2, 0, 2], [0, 1, 2])
  decoder.set_rows([0, 0, 2], [0, 1, 2])


def test_a_whole_sequence_is_not_read_behind_a_prefix(decoder, monkeypatch):
  monkeypatch.setattr(decoder, "_prefill_chunk", lambda ids, slot, p0: None)
  decoder.prefill([1] * 80, slot=0)
  decoder.prefill([1] * 70, slot=3)
  decoder.share_prefix(3, 70)
  with pytest.raises(ValueError, match="slot 0 holds what follows 0 places of a prefix, not 70"): decoder.set_rows([80, 70, 70], [0, 1, 2])
  decoder.set_rows([75, 75, 75], [1, 1, 2])           # (slots filled by nobody here: what they hold is the program's)
  decoder.share_prefix()
  decoder.set_rows([80, 5, 5], [0, 1, 2])
  decoder.share_prefix(3, 70)
  decoder.set_rows([70, 75, 75], [0, 1, 2])           # (slot 0 anew, behind the prefix)
  decoder.share_prefix()
  with pytest.raises(ValueError, match="slot 0"): decoder.prefill([1], slot=0, p0=6)
  decoder.prefill([1], slot=0)
  decoder.prefill([1], slot=0, p0=1)


def test_heads_that_packed_attention_does_not_take_are_refused_before_any_key_is_put(decoder, monkeypatch):
  def launched(T): raise AssertionError("past the checks")
  monkeypatch.setattr(decoder, "_prefill_buffers", launched)
  decoder.hd = 32
  with pytest.raises(NotImplementedError, match="head_dim"): decoder.prefill_batch([[1, 2]])
  with pytest.raises(NotImplementedError, match="head_dim"): decoder.share_prefix(3, 70)
  assert (decoder.behind == -1).all() and decoder.prefix_slot is None


def test_the_captured_step_stays_where_only_the_counts_change(decoder, monkeypatch):
  # a request with another count: the step's kernels read it when they run; another length, or an end, is another capture, which
  # waits for a replay that may be running
  waited = []
  monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: waited.append(device))
  for share, kept in (((3, 70), False), ((3, 70, [70, 0, 35]), True), ((2, 70), True), ((2, 64), False), ((), False), ((), True)):
    decoder.graph = graph = object()
    waited.clear()
    decoder.share_prefix(*share)
    assert (decoder.graph is graph) == kept and (decoder.graph is None) == (not kept) and len(waited) == (not kept), share
    assert not decoder.placed and decoder.prefix_row.item() == (share[0] if share else 0) * 100

"""The workspaces of many sequences' attention: a size taken for some rows, heads and bounds holds every call of no more of each
(a service takes one for its largest batch), and what the sizes are."""
import random
import pytest
import torch
from ferrite_amd import lib

pytestmark = pytest.mark.skipif(not lib.PATH.exists(), reason="libferrite_hip.so not built")


def log(rng, lo, hi):
  return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def test_packed_sizes_grow_with_every_argument():
  size, rng = lib.load().fh_attention_packed_workspace_bytes, random.Random(1)
  for _ in range(20000):
    kv, rep, hd = rng.choice([1, 2, 3, 8, 32]), rng.choice([1, 3, 4, 8]), rng.choice([64, 128])
    rows, n, ctx = log(rng, 1, 20000), log(rng, 1, 300), log(rng, 1, 70000)
    most = size(rows, n, kv * rep, kv, hd, ctx)
    for r, m, c in ((log(rng, 1, rows), log(rng, 1, n), log(rng, 1, ctx)), (log(rng, 1, rows), n, ctx), (rows, 1, ctx), (rows, n, log(rng, 1, ctx))):
      assert size(r, m, kv * rep, kv, hd, c) <= most, (r, m, c, rows, n, ctx, kv, rep, hd)
  # the service's sizes: 8192 rows in 16 prompts hold 200 rows of one
  assert size(8192, 16, 32, 8, 128, 4096) >= size(200, 1, 32, 8, 128, 4096) >= 16640000


def test_shared_sizes_grow_with_every_argument():
  size, rng = lib.load().fh_attention_shared_workspace_bytes, random.Random(2)
  for _ in range(20000):
    kv, rep, hd = rng.choice([1, 2, 3, 8, 32]), rng.choice([1, 3, 4, 8]), rng.choice([64, 128])
    batch, pre, own = log(rng, 1, 300), log(rng, 1, 70000) - 1, log(rng, 1, 70000) - 1
    most = size(batch, kv * rep, kv, hd, pre, own)
    for b, p, o in ((log(rng, 1, batch), log(rng, 1, pre + 1) - 1, log(rng, 1, own + 1) - 1), (1, pre, own), (batch, 0, own), (batch, pre, 0), (batch, pre, own // 2)):
      assert size(b, kv * rep, kv, hd, p, o) <= most, (b, p, o, batch, pre, own, kv, rep, hd)


def test_exact_sizes():
  pk, sh = lib.load().fh_attention_packed_workspace_bytes, lib.load().fh_attention_shared_workspace_bytes
  part = lambda hd: 4 * (hd + 2)
  assert pk(60, 3, 9, 3, 64, 64) == 0                                          # (one tile of keys: never split)
  assert pk(60, 3, 9, 3, 64, 65) == 60 * 9 * 2 * part(64)
  assert pk(10, 1, 8, 2, 128, 1 << 20) == 10 * 8 * 32 * part(128)
  assert pk(1 << 20, 64, 32, 8, 128, 1 << 20) == 3 * 128 * 256 * part(128)     # (many pairs: the most that any sizes split)
  assert sh(1, 8, 2, 64, 0, 0) == 8 * 2 * part(64)                             # (a part of the prefix, one of the row's own)
  assert sh(4, 9, 3, 64, 180, 40) == 4 * 9 * (3 + 1) * part(64)
  assert sh(64, 32, 8, 128, 16384, 700) == 64 * 32 * (32 + 11) * part(128)
  assert sh(5000, 32, 8, 128, 16384, 700) == 5000 * 32 * 2 * part(128)


def test_a_workspace_too_small_is_refused():
  # (before any launch)
  import test_sequences_refusals as R
  with pytest.raises(ValueError, match="fh_attention_packed_workspace_bytes"): R.packed(ctx=100000, len=100000)
  with pytest.raises(ValueError, match="fh_attention_packed_workspace_bytes"): R.packed(ctx=100000, len=100000, ws=R.P, wb=10 * 8 * 2 * 66 * 4 - 1)
  with pytest.raises(ValueError, match="fh_attention_shared_workspace_bytes"): R.shared(ws=R.P, wb=4 * 8 * 2 * 66 * 4 - 1)
  with pytest.raises(ValueError, match="fh_attention_shared_workspace_bytes"): R.shared(ws=R.P + 8, wb=1 << 30)


@pytest.mark.skipif(torch.cuda.is_available(), reason="(a call that is not refused would launch on the host's pointers)")
@pytest.mark.parametrize("batch,prefix,own,parts", [(16, 200, 4096, 4 + 2), (16, 4096, 8192, 16 + 2)])
def test_many_own_keys_behind_a_short_prefix_are_split(batch, prefix, own, parts):
  # (what the smallest accepted workspace says of the parts: one part less than these is refused)
  import test_sequences_refusals as R
  with pytest.raises(ValueError, match="fh_attention_shared_workspace_bytes"):
    R.shared(batch=batch, heads=32, kv=8, hd=128, len=100000, mp=prefix, mo=own, ws=R.P, wb=batch * 32 * parts * 4 * 130 - 1)

"""What the attention of many sequences and the logit rules refuse, on the host before any launch (no GPU needed: every
call here fails its checks), and their workspaces' sizes."""
import ctypes
import pytest
import torch
from ferrite_amd import lib, ops

needs_lib = pytest.mark.skipif(not lib.PATH.exists(), reason="libferrite_hip.so not built")
BUF = ctypes.create_string_buffer(1 << 12)
P = (ctypes.addressof(BUF) + 63) // 64 * 64


def packed(**kw):
  a = dict(q=P, qd=lib.F32, ldq=512, cache=P, cd=lib.BF16, len=100, rows=10, n=2, heads=8, kv=2, hd=64, starts=P, p0=P, first=P, prefix=None, shared=None,
           ctx=50, o=P, od=lib.BF16, ldo=512, ws=None, wb=0) | kw
  return lib.call("fh_attention_prefill_packed", *a.values(), None)


def shared(**kw):
  a = dict(q=P, qd=lib.F32, cache=P, cd=lib.BF16, len=100, batch=4, heads=8, kv=2, hd=64, places=P, first=P, prefix=P, shared=P, mp=50, mo=20, o=P,
           od=lib.BF16, ws=None, wb=0) | kw
  return lib.call("fh_attention_decode_shared", *a.values(), None)


def rules(**kw):
  a = dict(x=P, ldl=64, rows=2, vocab=64, tokens=None, ldt=0, most=0, lengths=None, prompts=None, rep=None, pre=None, fre=None, ids=None, bias=None, ldb=0,
           nb=0, allowed=None, ldm=0, out=P + 1024, ldo=64) | kw
  return lib.call("fh_logit_rules", *a.values(), None)


@needs_lib
@pytest.mark.parametrize("kw,err", [
  (dict(q=None), ValueError), (dict(starts=None), ValueError), (dict(o=None), ValueError), (dict(rows=0), ValueError), (dict(n=0), ValueError),
  (dict(heads=7), ValueError), (dict(hd=96), NotImplementedError), (dict(hd=256, ldq=2048, ldo=2048), NotImplementedError), (dict(qd=lib.BFP8), ValueError), (dict(cd=lib.I32), NotImplementedError),
  (dict(od=lib.BF16_T16), ValueError), (dict(ldq=510), ValueError), (dict(ldq=256), ValueError), (dict(ldo=500), ValueError), (dict(q=P + 4), ValueError),
  (dict(cache=P + 8), ValueError), (dict(o=P + 4), ValueError), (dict(ctx=0), ValueError), (dict(shared=P), ValueError), (dict(prefix=P), ValueError),
  (dict(len=0), ValueError), (dict(rows=1 << 31), ValueError), (dict(len=1 << 30), NotImplementedError), (dict(rows=1 << 29), NotImplementedError)])
def test_packed_refuses(kw, err):
  lib.load()
  with pytest.raises(err, match="fh_attention_prefill_packed"): packed(**kw)


@needs_lib
@pytest.mark.parametrize("kw,err", [
  (dict(q=None), ValueError), (dict(places=None), ValueError), (dict(shared=None), ValueError), (dict(prefix=None), ValueError), (dict(batch=0), ValueError),
  (dict(heads=7), ValueError), (dict(hd=32), NotImplementedError), (dict(od=lib.BFP4), ValueError), (dict(mp=-1), ValueError), (dict(mo=-1), ValueError),
  (dict(cd=9), NotImplementedError), (dict(qd=9), ValueError), (dict(cache=P + 2), ValueError)])
def test_shared_refuses(kw, err):
  lib.load()
  with pytest.raises(err, match="fh_attention_decode_shared"): shared(**kw)


@needs_lib
@pytest.mark.parametrize("kw,err", [
  (dict(x=None), ValueError), (dict(out=None), ValueError), (dict(rows=0), ValueError), (dict(ldl=63), ValueError), (dict(ldo=63), ValueError),
  (dict(out=P, ldo=65), ValueError), (dict(lengths=P), ValueError), (dict(tokens=P, ldt=3, most=4), ValueError), (dict(ids=P), ValueError),
  (dict(ids=P, bias=P, ldb=4, nb=5), ValueError), (dict(ids=P, bias=P, ldb=2000, nb=1025), NotImplementedError), (dict(allowed=P, ldm=1), ValueError),
  (dict(rows=65536), NotImplementedError), (dict(tokens=P, ldt=1 << 30, most=1 << 30), NotImplementedError)])
def test_rules_refuse(kw, err):
  lib.load()
  with pytest.raises(err, match="fh_logit_rules"): rules(**kw)


@needs_lib
def test_workspace_sizes():
  lib.load()
  pk, sh = lib.load().fh_attention_packed_workspace_bytes, lib.load().fh_attention_shared_workspace_bytes
  assert pk(0, 1, 8, 2, 64, 100) == 0 and pk(10, 0, 8, 2, 64, 100) == 0 and pk(10, 1, 7, 2, 64, 100) == 0 and pk(10, 1, 8, 2, 64, 0) == 0
  assert sh(0, 8, 2, 64, 100, 100) == 0 and sh(4, 7, 2, 64, 100, 100) == 0 and sh(4, 8, 2, 64, -1, 100) == 0
  # (what a call needs grows no further than a bound its caller can rely on: a part a split, 2^31 rows apart from none)
  assert 0 <= pk(1 << 20, 64, 32, 8, 128, 1 << 20) < 1 << 40 and 0 <= sh(256, 32, 8, 128, 1 << 20, 1 << 20) < 1 << 36


def test_python_refuses_what_is_not_on_the_gpu_or_misshapen():
  # (the shape checks come before any device work, the device checks before the call)
  i = lambda n: torch.zeros(n, dtype=torch.int32)
  q, c = torch.zeros(4, 128), torch.zeros(2, 20, 64)
  with pytest.raises(ValueError, match="on the GPU"): ops.attention_prefill_packed(q, c, 2, 1, 64, i(2), i(1), i(1), 10)
  with pytest.raises(ValueError, match="on the GPU"): ops.attention_decode_shared(q, c, 2, 1, 64, i(4), i(4), i(1), i(4), 10, 10)
  with pytest.raises(ValueError, match="on the GPU"): ops.logit_rules(q)

"""What the operators over a cache in pages and the low-rank adapters refuse, on the host before any launch (no GPU needed: every call
here fails its checks), and their workspaces' sizes."""
import copy, ctypes, pickle
import pytest
import torch
from ferrite_amd import lib, ops

needs_lib = pytest.mark.skipif(not lib.PATH.exists(), reason="libferrite_hip.so not built")
BUF = ctypes.create_string_buffer(1 << 12)
P = (ctypes.addressof(BUF) + 63) // 64 * 64


def attend(**kw):
  a = dict(q=P, qd=lib.F32, ldq=512, cache=P, cd=lib.BF16, len=96, rows=10, n=2, heads=8, kv=2, hd=64, starts=P, p0=P, tables=P, ldt=6, cols=6, page=16, ctx=90,
           o=P, od=lib.BF16, ldo=512, ws=None, wb=0) | kw
  return lib.call("fh_attention_paged", *a.values(), None)


def append(**kw):
  a = dict(x=P, xd=lib.F32, ldx=768, rows=10, n=2, heads=8, kv=2, hd=64, qn=None, kn=None, eps=1e-5, centered=0, cos=P, sin=P, turns=9, starts=P, p0=P, tables=P,
           ldt=6, cols=6, page=16, q=P, qd=lib.F32, ldq=512, cache=P, cd=lib.BF16, len=96) | kw
  return lib.call("fh_rope_append_paged", *a.values(), None)


def lora(**kw):
  a = dict(x=P, xd=lib.F32, ldx=64, rows=4, K=64, a=P, b=P, wd=lib.BF16, n=2, rank=8, parts=2, cols=(32, 16), scale=None, ids=P, res=P, ldr=48, y=P, yd=lib.F32, ldy=48,
           ws=P, wb=1 << 20) | kw
  if a["cols"] is not None: a["cols"] = (ctypes.c_int64 * len(a["cols"]))(*a["cols"])
  return lib.call("fh_lora", *a.values(), None)


@needs_lib
@pytest.mark.parametrize("kw,err", [
  (dict(q=None), ValueError), (dict(starts=None), ValueError), (dict(p0=None), ValueError), (dict(tables=None), ValueError), (dict(o=None), ValueError), (dict(rows=0), ValueError),
  (dict(n=0), ValueError), (dict(heads=7), ValueError), (dict(hd=96), NotImplementedError), (dict(qd=lib.BFP8), ValueError), (dict(cd=lib.I32), NotImplementedError),
  (dict(od=lib.BF16_T16), ValueError), (dict(ldq=510), ValueError), (dict(ldq=256), ValueError), (dict(ldo=500), ValueError), (dict(q=P + 4), ValueError),
  (dict(cache=P + 8), ValueError), (dict(o=P + 4), ValueError), (dict(ctx=0), ValueError), (dict(page=8), NotImplementedError), (dict(page=48), NotImplementedError),
  (dict(page=0), NotImplementedError), (dict(page=64), ValueError), (dict(len=0), ValueError), (dict(len=100), ValueError), (dict(cols=0), ValueError), (dict(ldt=5), ValueError),
  (dict(rows=1 << 31), ValueError), (dict(len=1 << 30), NotImplementedError), (dict(rows=1 << 29), NotImplementedError),
  (dict(len=16000, cols=1000, ldt=1000, ctx=16000), ValueError)])
def test_attention_refuses(kw, err):
  lib.load()
  with pytest.raises(err, match="fh_attention_paged"): attend(**kw)  # (the last: its workspace is missing)


@needs_lib
@pytest.mark.parametrize("kw,err", [
  (dict(x=None), ValueError), (dict(q=None), ValueError), (dict(cache=None), ValueError), (dict(tables=None), ValueError), (dict(rows=0), ValueError), (dict(rows=1 << 31), ValueError),
  (dict(n=0), ValueError), (dict(heads=0), ValueError), (dict(kv=0), ValueError), (dict(hd=96), NotImplementedError), (dict(xd=lib.BFP8), ValueError), (dict(qd=lib.BF16_T16), ValueError),
  (dict(cd=lib.I32), NotImplementedError), (dict(sin=None), ValueError), (dict(turns=0), ValueError), (dict(page=8), NotImplementedError), (dict(page=64), ValueError),
  (dict(len=8), ValueError), (dict(len=1 << 30), NotImplementedError), (dict(cols=0), ValueError), (dict(ldt=5), ValueError), (dict(ldx=767), ValueError), (dict(ldx=764), ValueError),
  (dict(ldq=510), ValueError), (dict(x=P + 4), ValueError), (dict(q=P + 4), ValueError), (dict(cache=P + 8), ValueError), (dict(qn=P + 4), ValueError), (dict(cos=P + 8), ValueError),
  (dict(), ValueError), (dict(ldq=768, qd=lib.BF16), ValueError), (dict(ldq=768, rows=1 << 25), NotImplementedError)])
def test_append_refuses(kw, err):
  lib.load()
  with pytest.raises(err, match="fh_rope_append_paged"): append(**kw)  # (the last but two: q in qkv's columns with rows of its own)


@needs_lib
@pytest.mark.parametrize("kw,err", [
  (dict(x=None), ValueError), (dict(a=None), ValueError), (dict(b=None), ValueError), (dict(cols=None), ValueError), (dict(ids=None), ValueError), (dict(y=None), ValueError),
  (dict(rows=0), ValueError), (dict(K=0), ValueError), (dict(n=0), ValueError), (dict(rows=(64 * 65535) + 1), NotImplementedError), (dict(K=60), NotImplementedError),
  (dict(rank=12), NotImplementedError), (dict(rank=136), NotImplementedError), (dict(rank=0), NotImplementedError), (dict(parts=0), NotImplementedError),
  (dict(parts=5, cols=(8,) * 5), NotImplementedError), (dict(cols=(32, 12)), NotImplementedError), (dict(cols=(32, 0)), NotImplementedError),
  (dict(cols=(1 << 29, 1 << 29)), NotImplementedError), (dict(xd=lib.BFP8), ValueError), (dict(wd=lib.BFP8), ValueError), (dict(yd=lib.BF16_T16), ValueError),
  (dict(ldx=56), ValueError), (dict(ldx=66), ValueError), (dict(ldy=40), ValueError), (dict(ldy=50), ValueError), (dict(ldr=44), ValueError), (dict(ldr=52), ValueError),
  (dict(x=P + 8), ValueError), (dict(b=P + 8), ValueError), (dict(y=P + 8, res=None), ValueError), (dict(ws=None), ValueError), (dict(wb=16), ValueError), (dict(ws=P + 8), ValueError),
  (dict(), ValueError)])
def test_lora_refuses(kw, err):
  lib.load()
  with pytest.raises(err, match="fh_lora"): lora(**kw)  # (the last: y is x)


@needs_lib
@pytest.mark.parametrize("kw,err", [
  (dict(x=None), ValueError), (dict(y=None), ValueError), (dict(rows=0), ValueError), (dict(split=0), ValueError), (dict(xd=lib.BFP8), ValueError), (dict(yd=lib.BF16_T16), ValueError),
  (dict(split=12), NotImplementedError), (dict(ldx=60), ValueError), (dict(ldx=66), ValueError), (dict(ldy=28), ValueError), (dict(ldy=34), ValueError), (dict(x=P + 8), ValueError),
  (dict(y=P + 8), ValueError), (dict(rows=1 << 40), NotImplementedError)])
def test_silu_gate_refuses(kw, err):
  lib.load()
  a = dict(x=P, xd=lib.F32, ldx=64, rows=4, split=32, y=P + 1024, yd=lib.F32, ldy=32) | kw
  with pytest.raises(err, match="fh_silu_gate_rows"): lib.call("fh_silu_gate_rows", *a.values(), None)


@needs_lib
def test_workspace_sizes():
  L = lib.load()
  pg, lo = L.fh_attention_paged_workspace_bytes, L.fh_lora_workspace_bytes
  assert pg(0, 1, 8, 2, 64, 100) == 0 and pg(10, 0, 8, 2, 64, 100) == 0 and pg(10, 1, 7, 2, 64, 100) == 0 and pg(10, 1, 8, 2, 64, 0) == 0
  assert 0 <= pg(1 << 20, 64, 32, 8, 128, 1 << 20) < 1 << 40
  assert lo(0, 64, 8, 1) == 0 and lo(4, 0, 8, 1) == 0 and lo(4, 64, 0, 1) == 0 and lo(4, 64, 136, 1) == 0 and lo(4, 64, 8, 5) == 0
  # one for some rows (or context, or sequences) serves every call of no more
  sizes = [lo(rows, 4096, 16, 3) for rows in range(1, 40000, 7)]
  assert sizes == sorted(sizes)
  for args in ((300, 8, 32, 8, 128), (64, 64, 32, 8, 128), (9, 9, 4, 1, 64)):
    for most in (1, 64, 100, 3000, 100000):
      top = pg(*args, most)
      assert all(pg(rows, n, heads, args[3], args[4], c) <= top for rows in (1, args[0] // 2, args[0]) for n in (1, args[1]) for heads in (args[3], args[2])
                 for c in (1, 65, 2000, most) if c <= most)


def test_python_refuses_what_is_not_on_the_gpu_or_misshapen():
  i = lambda *n: torch.zeros(*n, dtype=torch.int32)
  q, c = torch.zeros(4, 128), torch.zeros(2, 32, 64)
  with pytest.raises(ValueError, match="on the GPU"): ops.attention_paged(q, c, 2, 1, 64, i(2), i(1), i(1, 2), 16, 10)
  with pytest.raises(ValueError, match="on the GPU"): ops.rope_append_paged(torch.zeros(4, 256), c, 2, 1, 64, None, None, i(2), i(1), i(1, 2), 16)
  with pytest.raises(ValueError, match="on the GPU"): ops.lora(q, ops.Adapters(torch.zeros(1, 8, 128), torch.zeros(1, 8, 8), None, (8,)), i(4))
  with pytest.raises(ValueError, match="parts"): ops.lora(q, ops.Adapters(torch.zeros(1, 8, 128), torch.zeros(1, 8, 8), None, (16,)), i(4))
  with pytest.raises(ValueError, match="alike"): ops.lora(q, ops.Adapters(torch.zeros(1, 8, 128), torch.zeros(1, 8, 8, dtype=torch.bfloat16), None, (8,)), i(4))


def test_a_copy_of_adapters_has_sizes_of_its_own():
  # (a call passes the parts' address: a copy's must outlive the adapters that it was made from)
  ad = ops.Adapters(torch.zeros(2, 16, 64), torch.zeros(2, 24, 8), None, (16, 8))
  for other in (copy.copy(ad), copy.deepcopy(ad), pickle.loads(pickle.dumps(ad))):
    cols = other._call[4]
    assert other.parts == ad.parts and tuple(cols) == (16, 8) and cols is not ad._call[4]
    assert other._call[3][4] == ctypes.addressof(cols) != ad._call[3][4]

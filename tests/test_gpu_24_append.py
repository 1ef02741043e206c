"""The heads' norms, rotation and put into a cache in pages (fh_rope_append_paged) against the formula in 64 bits: every type and format,
ragged rows, places and pages outside, strides, rows and cache rows that are nobody's, captured calls. Errors are bounded by the roundings:
a head's mean of squares is a sum of hd squares in a tree at most 12 additions deep and a root and a quotient after it, each value
three products and a sum more: 24 2^-24 of |n0 cos| + |n1 sin|; then the output's own rounding, half a step (bf16 2^-8); a block float's
value is off by its bf16 rounding and at most a step of its run (half, and a whole one where it saturates)."""
import numpy as np
import pytest
import torch
from oracle import bfp as O

pytestmark = pytest.mark.gpu
DTYPE = {"fp32": torch.float32, "bf16": torch.bfloat16}


def ops():
  from ferrite_amd import ops as m
  return m


def ints(v):
  return torch.tensor(v, dtype=torch.int32, device="cuda")


def values_of(cache, planes, rows, hd):
  """A cache's values in float64."""
  if isinstance(cache, torch.Tensor): return cache.double().cpu()
  raw = cache.data.cpu().numpy()
  n = planes * rows * hd
  if cache.fmt == "bfp8": q, bias = raw[:n].view(np.int8).astype(np.int64), 133
  else:
    b = raw[:n // 2].astype(np.int64)
    q, bias = np.stack([b & 15, b >> 4], 1).reshape(-1), 129
    q = np.where(q > 7, q - 16, q)
  e = raw[-(n // 16):].astype(np.int64).repeat(16)
  return torch.from_numpy(q * 2.0 ** (e - bias)).view(planes, rows, hd)


def case(seed, heads, kv, hd, lens, before, page=16, x="fp32", fmt="bf16", q="fp32", norm=True, centered=False, turn=True, ahead=0, pad=0, wide=0, places=None):
  rng = np.random.default_rng(seed)
  n, T = len(lens), max(1, ahead + sum(lens) + pad)
  counts = [-(-(a + b) // page) for a, b in zip(lens, before)]
  ids, at, cols = rng.permutation(sum(counts) + 2), 0, max(1, max(counts))
  tables = np.full((n, cols + 2), 1 << 30)
  for i, c in enumerate(counts):
    tables[i, :c] = ids[at:at + c]
    at += c
  rows = len(ids) * page
  starts = ahead + np.concatenate([[0], np.cumsum(lens)])
  H = heads + 2 * kv
  xb = torch.from_numpy(rng.normal(0, 2, (T, H * hd + wide)).astype(np.float32)).to(DTYPE[x])
  most = places or max(1, max(a + b for a, b in zip(lens, before)))
  ang = np.arange(most)[:, None] * 10000.0 ** (-np.arange(0, hd, 2) / hd)
  cos, sin = (torch.from_numpy(O.bf16(np.concatenate([f(ang)] * 2, 1).astype(np.float32))) for f in (np.cos, np.sin))
  w = [torch.from_numpy(rng.normal(1, 0.2, hd).astype(np.float32)) if norm else None for _ in range(2)]
  cache = ops().kv_cache(2 * kv, rows, hd, fmt)
  data = cache.data if fmt in ("bfp8", "bfp4") else cache
  if fmt in DTYPE: data.fill_(3.0)
  else: data.fill_(0x55)
  old = values_of(cache, 2 * kv, rows, hd)
  qb = torch.full((T, heads * hd + wide), 7.0, dtype=DTYPE[q], device="cuda")
  dev = lambda t: None if t is None else t.cuda()
  got = ops().rope_append_paged(xb.cuda()[:, :H * hd], cache, heads, kv, hd, dev(cos) if turn else None, dev(sin) if turn else None, ints(starts), ints(before),
                                ints(tables)[:, :cols], page, q_norm=dev(w[0]), k_norm=dev(w[1]), eps=1e-5, centered=centered, q=qb[:, :heads * hd])
  held = values_of(cache, 2 * kv, rows, hd)
  # the formula
  want_q, tol_q = torch.full((T, heads * hd), 7.0, dtype=torch.float64), torch.zeros(T, heads * hd, dtype=torch.float64)
  want, tol = old.clone(), torch.zeros_like(old)
  for s in range(n):
    for i in range(lens[s]):
      t, p = int(starts[s]) + i, before[s] + i
      y = xb[t, :H * hd].double().view(H, hd)
      size = y.abs()
      tp = min(max(p, 0), most - 1)
      if norm:
        r = 1 / torch.sqrt((y * y).mean(1, keepdim=True) + np.float64(np.float32(1e-5)))
        wt = torch.cat([w[0].double().expand(heads, hd), w[1].double().expand(kv, hd)]) + (1 if centered else 0)
        y = torch.cat([y[:heads + kv] * r[:heads + kv] * wt, y[heads + kv:]])
        size = y.abs()
      if turn:
        c, sn, h2 = cos[tp].double(), sin[tp].double(), hd // 2
        k = y[:heads + kv]
        rot = torch.cat([-k[:, h2:], k[:, :h2]], 1)
        y = torch.cat([k * c + rot * sn, y[heads + kv:]])
        size = torch.cat([k.abs() * c.abs() + rot.abs() * sn.abs(), size[heads + kv:]])
      err = 24 * 2.0 ** -24 * size
      want_q[t] = y[:heads].reshape(-1)
      tol_q[t] = (err[:heads] + (2.0 ** -8 * y[:heads].abs() if q == "bf16" else 0)).reshape(-1)
      if p < 0 or p // page >= cols or not 0 <= tables[s, p // page] < len(ids): continue
      row, v, e = tables[s, p // page] * page + p % page, y[heads:], err[heads:]
      want[:, row] = v
      if fmt == "fp32": tol[:, row] = e
      elif fmt == "bf16": tol[:, row] = e + 2.0 ** -8 * v.abs()
      else:
        top = torch.frexp((v.abs() + e).view(2 * kv, hd // 16, 16).amax(2) * (1 + 2.0 ** -8)).exponent  # (2^(top - 1) <= the largest)
        step = 2.0 ** (top - (7 if fmt == "bfp8" else 3)).double()
        tol[:, row] = e + 2.0 ** -8 * v.abs() + step.repeat_interleave(16, 1)
  assert (qb[:, heads * hd:] == 7).all()
  return got, want_q, tol_q, held, want, tol


def check(r, what):
  got, want_q, tol_q, held, want, tol = r
  bad = (got.double().cpu() - want_q).abs() > tol_q
  assert not bad.any(), (what, "q", int(bad.sum()))
  bad = (held - want).abs() > tol
  assert not bad.any() and torch.isfinite(held).all(), (what, "cache", int(bad.sum()))


@pytest.mark.parametrize("lens,before,page", [([1], [0], 16), ([1], [16], 16), ([1, 1, 1], [15, 100, 0], 32), ([5, 0, 33, 1], [0, 4, 14, 63], 16), ([70, 3], [9, 126], 128)])
@pytest.mark.parametrize("heads,kv,hd,x,fmt,q", [(9, 3, 64, "fp32", "bf16", "fp32"), (8, 2, 128, "bf16", "bfp8", "bf16"), (4, 4, 64, "fp32", "fp32", "fp32"),
                                                 (1, 1, 64, "bf16", "bfp4", "fp32"), (3, 1, 128, "fp32", "bfp4", "bf16"), (32, 8, 128, "bf16", "bf16", "bf16")])
def test_append(cuda, lens, before, page, heads, kv, hd, x, fmt, q):
  print(f"append {lens} {before} {page} {heads}/{kv} {hd} {x} {fmt} {q}", flush=True)
  check(case(1, heads, kv, hd, lens, before, page, x, fmt, q), (lens, fmt))


@pytest.mark.parametrize("fmt", ["fp32", "bf16", "bfp8", "bfp4"])
@pytest.mark.parametrize("norm,centered,turn", [(False, False, True), (True, True, True), (True, False, False)])
def test_append_forms(cuda, fmt, norm, centered, turn):
  print(f"append forms {fmt} {norm} {centered} {turn}", flush=True)
  for hd, x, q in ((64, "bf16", "fp32"), (128, "fp32", "bf16")):
    check(case(2, 6, 2, hd, [7, 20], [40, 3], 16, x, fmt, q, norm, centered, turn), (fmt, hd))


def test_append_strides_and_rows_behind(cuda):
  r = case(3, 6, 2, 64, [4, 0, 9], [30, 2, 16], ahead=3, pad=6, wide=16)
  check(r, "strides")
  assert (r[0][:3] == 7).all() and (r[0][16:] == 7).all()


def test_append_many_heads_and_sequences(cuda):
  # more lanes than a workgroup's 1024 (heads in rounds); more sequences than a wave looks through at once
  check(case(4, 150, 5, 64, [3, 1], [0, 40], fmt="bfp8"), "heads")
  rng = np.random.default_rng(5)
  for n in (64, 65, 140):
    lens = [int(i) for i in rng.integers(0, 4, n)]
    lens[-1], lens[63] = 2, 0
    check(case(5, 2, 1, 64, lens, [int(i) for i in rng.integers(0, 60, n)], pad=2), n)


def test_append_places_outside(cuda):
  # places behind the rotation's tables read the nearest row; places below 0 or past the sequence's table, and pages outside the
  # cache, write nothing
  check(case(6, 4, 2, 64, [10, 4], [20, 0], places=13), "few places")
  check(case(7, 4, 2, 64, [10, 4], [-6, 0]), "below 0")
  rng = np.random.default_rng(8)
  x = torch.from_numpy(rng.normal(0, 1, (6, 4 * 64)).astype(np.float32)).cuda()
  for tables, p0, wrote in (([[1 << 30], [-1]], [0, 0], []), ([[0], [1]], [16, 1 << 30], []), ([[2], [1]], [14, -2], [46, 47, 16])):
    cache = torch.full((2, 48, 64), 3.0, device="cuda")
    ops().rope_append_paged(x, cache, 2, 1, 64, None, None, ints([0, 3, 6]), ints(p0), ints(tables), 16)
    changed = (cache != 3.0).any(2).any(0).cpu().nonzero()[:, 0].tolist()
    assert changed == sorted(wrote), (tables, changed)


@pytest.mark.parametrize("fmt", ["bfp8", "bfp4", "bf16"])
def test_append_rounds_as_the_oracle(cuda, fmt):
  # neither normed nor turned: the cache holds the bits that the oracle's rounding gives
  rng = np.random.default_rng(9)
  for hd in (64, 128):
    x = (rng.normal(0, 1, (20, 5 * hd)) * np.exp(rng.normal(0, 3, (20, 5 * hd)))).astype(np.float32)
    x[3], x[4, ::7] = 0, 0
    cache = ops().kv_cache(4, 32, hd, fmt)
    q = ops().rope_append_paged(torch.from_numpy(x).cuda(), cache, 1, 2, hd, None, None, ints([0, 20]), ints([5]), ints([[1, 0]]), 16)
    assert torch.equal(q.cpu(), torch.from_numpy(x[:, :hd]))
    rows = np.concatenate([np.arange(21, 32), np.arange(0, 9)])
    held = values_of(cache, 4, 32, hd)[:, rows]
    kv = x[:, hd:].reshape(20, 4, hd).transpose(1, 0, 2)
    want = O.bfp_values(*O.bfp_parts(kv, fmt), fmt) if fmt != "bf16" else O.bf16(kv).astype(np.float64)
    assert np.array_equal(held.numpy(), want), (fmt, hd)


def test_append_past_32_bits(cuda):
  rows = 17 << 20
  cache = torch.zeros(4, rows, 64, dtype=torch.bfloat16, device="cuda")
  x = torch.randn(5, 4 * 64 + 64, device="cuda")
  ops().rope_append_paged(x, cache, 1, 2, 64, None, None, ints([0, 5]), ints([14]), ints([[rows // 16 - 2, rows // 16 - 1]]), 16)
  at = torch.tensor([rows - 18, rows - 17, rows - 16, rows - 15, rows - 14], device="cuda")
  assert torch.equal(cache[:, at], x[:, 64:].view(5, 4, 64).transpose(0, 1).to(torch.bfloat16))
  assert float(cache[:, :rows - 18].abs().max()) == 0 and float(cache[:, rows - 13:].abs().max()) == 0


def test_append_graph_and_stream(cuda):
  # a captured call replays with what the arrays hold then; another stream gives the same bits
  rng = np.random.default_rng(10)
  x = torch.from_numpy(rng.normal(0, 1, (6, 8 * 64)).astype(np.float32)).cuda()
  ang = torch.from_numpy((np.arange(100)[:, None] * np.ones(64)).astype(np.float32))
  cos, sin = torch.cos(ang).cuda(), torch.sin(ang).cuda()
  starts, tables, p0 = ints([0, 1, 4, 6]), ints([[0, 1], [2, 3], [5, 4]]), ints([3, 15, 20])
  call = lambda cache, q: ops().rope_append_paged(x, cache, 4, 2, 64, cos, sin, starts, p0, tables, 16, q=q)
  new = lambda: (torch.zeros(4, 96, 64, device="cuda"), torch.zeros(6, 256, device="cuda"))
  (c1, q1), side = new(), torch.cuda.Stream()
  call(c1, q1)
  torch.cuda.synchronize()
  g = torch.cuda.CUDAGraph()
  with torch.cuda.graph(g): call(c1, q1)
  for spots, tabs in (([3, 15, 20], [[0, 1], [2, 3], [5, 4]]), ([0, 0, 30], [[1, 1], [0, 3], [2, 5]]), ([17, 2, 9], [[4, 5], [3, 2], [1, 0]])):
    p0.copy_(ints(spots))
    tables.copy_(ints(tabs))
    c1.zero_()
    g.replay()
    c2, q2 = new()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side): call(c2, q2)
    torch.cuda.synchronize()
    assert torch.equal(c1, c2) and torch.equal(q1, q2)


def test_append_in_place_and_many_rows(cuda):
  # q in qkv's own columns; rows of many sequences, several a workgroup, among them rows that are nobody's
  rng = np.random.default_rng(11)
  T, lens = 3333, [1] * 40 + [700, 0, 1300] + [3] * 20 + [900]
  starts = np.concatenate([[7], 7 + np.cumsum(lens)])
  before = rng.integers(0, 90, len(lens))
  counts = [-(-(a + int(b)) // 16) for a, b in zip(lens, before)]
  ids, at, tables = rng.permutation(sum(counts)), 0, np.full((len(lens), max(counts)), -1)
  for i, c in enumerate(counts):
    tables[i, :c] = ids[at:at + c]
    at += c
  x = torch.from_numpy(rng.normal(0, 1, (T, 8 * 64)).astype(np.float32)).cuda()
  ang = torch.from_numpy(rng.normal(0, 1, (1400, 64)).astype(np.float32)).cuda()
  args = (4, 2, 64, torch.cos(ang), torch.sin(ang), ints(starts), ints(before), ints(tables), 16)
  c1, c2 = (torch.zeros(4, 16 * len(ids), 64, device="cuda") for _ in range(2))
  want = ops().rope_append_paged(x, c1, *args, q=torch.full((T, 256), 7.0, device="cuda"))
  y = x.clone()
  ops().rope_append_paged(y, c2, *args, q=y[:, :256])
  used = slice(7, int(starts[-1]))
  assert torch.equal(y[used, :256], want[used]) and torch.equal(y[:, 256:], x[:, 256:]) and torch.equal(c1, c2)
  assert torch.equal(y[:7], x[:7]) and torch.equal(y[starts[-1]:], x[starts[-1]:]) and (want[:7] == 7).all() and (want[starts[-1]:] == 7).all()
  # v's rows are at their places, bit for bit
  for s in (0, 40, 42, 50, len(lens) - 1):
    p = int(before[s]) + np.arange(lens[s])
    rows = torch.from_numpy(tables[s, p // 16] * 16 + p % 16).cuda()
    assert torch.equal(c1[2:, rows].transpose(0, 1).reshape(lens[s], 128), x[starts[s]:starts[s + 1], 384:])

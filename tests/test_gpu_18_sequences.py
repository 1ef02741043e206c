"""Attention of many sequences at once (fh_attention_prefill_packed, fh_attention_decode_shared) against the formula in 64
bits within a bound derived from each rounding (seq_cases.attend): lengths of none, one and many, odd sizes, every cache
format, strides, prefixes shared by all, some or none, rows no request holds, values that no query may see, captured
calls, a workspace shared by two graphs."""
import numpy as np
import pytest
import torch
import seq_cases as S

pytestmark = pytest.mark.gpu


def ops():
  from ferrite_amd import ops as m
  return m


def ints(v):
  return torch.tensor(list(v), dtype=torch.int32, device="cuda")


def packed(seed, heads, kv, hd, lens, cached, prefix=0, fmt="bf16", q="fp32", o="bf16", before=0, pad=0, wide=0, spoil=None, slack=0):
  """A packed call and its oracle: (o, want, tol, rows of o that are no sequence's)."""
  rng = np.random.default_rng(seed)
  n, prefix_row, first, at = len(lens), 2, [], prefix + 3
  for a, c in zip(lens, cached):
    first.append(at)
    at += a + c + int(rng.integers(0, 4))
  cache, values = S.cache(rng, 2 * kv, at + 2, hd, fmt)
  T = before + sum(lens) + pad
  qb = torch.from_numpy(rng.normal(0, 1.5, (max(T, 1), heads * hd + wide)).astype(np.float32)).to(S.DTYPE[q])
  starts = before + np.concatenate([[0], np.cumsum(lens)])
  ob = torch.full((max(T, 1), heads * hd + wide), 7.0, dtype=S.DTYPE[o], device="cuda")
  if spoil: spoil(cache, first)
  qg, og = qb.cuda()[:, :heads * hd], ob[:, :heads * hd]
  shared = ints([prefix] * n) if prefix else None
  got = ops().attention_prefill_packed(qg, cache, heads, kv, hd, ints(starts), ints(prefix + c for c in cached), ints(first),
                                       prefix + max(a + c for a, c in zip(lens, cached)) + 1 + slack, prefix_row=ints([prefix_row]) if prefix else None, shared=shared, o=og)
  assert got.data_ptr() == og.data_ptr()
  want, tol = torch.full((T, heads * hd), 7.0, dtype=torch.float64), torch.zeros(T, heads * hd, dtype=torch.float64)
  for s in range(n):
    a, c = lens[s], cached[s]
    if not a: continue
    where = S.rows_of(prefix_row, prefix, first[s], prefix + c + a)
    lo = int(starts[s])
    want[lo:lo + a], tol[lo:lo + a] = S.attend(qb[lo:lo + a, :heads * hd], values, where, prefix + c + 1 + np.arange(a), kv, hd, o == "bf16")
  assert (ob[:, heads * hd:] == 7).all()  # (what lies between o's rows is not o's)
  return got, want, tol


@pytest.mark.parametrize("lens,cached,prefix", [
  ([1], [0], 0), ([20, 1, 30], [0, 0, 0], 0), ([64, 0, 63, 65], [0, 5, 1, 64], 0), ([129, 32, 31, 33], [0, 100, 17, 0], 0),
  ([5, 200], [300, 0], 70), ([1, 1, 1, 2], [63, 64, 65, 0], 1), ([0, 0, 3, 0], [4, 0, 0, 9], 128), ([260], [0], 0)])
@pytest.mark.parametrize("heads,kv,hd,fmt,q,o", [(9, 3, 64, "bf16", "fp32", "bf16"), (8, 2, 128, "bfp8", "fp32", "bf16"), (4, 4, 64, "fp32", "fp32", "fp32"),
                                                 (8, 1, 128, "bf16", "bf16", "fp32"), (6, 2, 128, "bfp4", "bf16", "bf16")])
def test_packed(cuda, lens, cached, prefix, heads, kv, hd, fmt, q, o):
  print(f"packed {lens} {cached} {prefix} {heads}/{kv} {hd} {fmt} {q} {o}", flush=True)
  got, want, tol = packed(1, heads, kv, hd, lens, cached, prefix, fmt, q, o)
  S.check(got, want, tol, (lens, fmt))


@pytest.mark.parametrize("fmt", ["bf16", "fp32", "bfp8", "bfp4"])
@pytest.mark.parametrize("hd,heads,kv", [(64, 16, 1), (128, 5, 5)])
@pytest.mark.parametrize("q,o", [("fp32", "fp32"), ("bf16", "bf16"), ("fp32", "bf16")])
def test_packed_types(cuda, fmt, hd, heads, kv, q, o):
  print(f"packed types {fmt} {hd} {heads}/{kv} {q} {o}", flush=True)
  got, want, tol = packed(2, heads, kv, hd, [70, 3, 11], [9, 0, 80], 40, fmt, q, o)
  S.check(got, want, tol, (fmt, hd, q, o))


def test_packed_strides_and_rows_behind(cuda):
  # rows before the first start and behind the last sequence keep what they held; q and o are columns of wider buffers
  got, want, tol = packed(3, 6, 2, 64, [40, 0, 25], [0, 0, 3], 0, before=5, pad=13, wide=24)
  S.check(got, want, tol, "strides")
  assert (got[:5] == 7).all() and (got[5 + 65:] == 7).all()


def test_packed_long_context_of_few_rows(cuda):
  # few rows after many cached ones (the keys' long axis), with the bound of the context far above what is there
  got, want, tol = packed(4, 8, 2, 128, [3, 40], [2000, 1111], 77, slack=3000)
  S.check(got, want, tol, "long")
  got, want, tol = packed(5, 3, 1, 64, [1, 2], [1500, 700], 0, fmt="fp32", o="fp32")
  S.check(got, want, tol, "long fp32")


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("fmt,o", [("bf16", "bf16"), ("fp32", "fp32"), ("bf16", "fp32")])
def test_packed_unseen_values(cuda, bad, fmt, o):
  # keys and values at places a row does not see (a later token's, another sequence's, rows of nobody) are NaN or infinite:
  # rows before them keep their results; rows that see them are not finite
  cut = 37  # (place 37 of the first sequence is spoilt: rows 0 .. 36 do not see it)
  def spoil(cache, first):
    cache[:, first[0] + cut] = bad
    cache[:, :2] = bad
    cache[:, -2:] = bad
  got, want, tol = packed(6, 4, 2, 64, [90, 20], [0, 4], 0, fmt, "fp32", o, spoil=spoil)
  S.check(got[:cut], want[:cut], tol[:cut], "before the place")
  S.check(got[90:], want[90:], tol[90:], "the other sequence")
  if bad != -float("inf"): assert not torch.isfinite(got[cut:90].float()).any(1).any() or bad == float("inf")
  assert not torch.isfinite(got[cut:90].float()).all(1).any()


def test_packed_past_32_bits(cuda):
  # a cache whose values lie past 2^31 elements: the last rows of the last plane
  rows, hd = 17 << 20, 64
  cache = torch.zeros(2, rows, hd, dtype=torch.bfloat16, device="cuda")
  rng = np.random.default_rng(7)
  some = torch.from_numpy(rng.normal(0, 1, (2, 50, hd)).astype(np.float32)).to(torch.bfloat16)
  cache[:, rows - 50:] = some.cuda()
  q = torch.from_numpy(rng.normal(0, 1, (30, 2 * hd)).astype(np.float32))
  for o in ("bf16", "fp32"):
    got = ops().attention_prefill_packed(q.cuda(), cache, 2, 1, hd, ints([0, 30]), ints([20]), ints([rows - 50]), 50, out_dtype=S.DTYPE[o])
    want, tol = S.attend(q, some.double(), torch.arange(50), 21 + np.arange(30), 1, hd, o == "bf16")
    S.check(got, want, tol, o)
    places = ints([49] * 2)
    got = ops().attention_decode_shared(q[:2].cuda(), cache, 2, 1, hd, places, ints([rows - 20] * 2), ints([rows - 50]), ints([30] * 2), 30, 20, out_dtype=S.DTYPE[o])
    want, tol = S.attend(q[:2], some.double(), torch.arange(50), [50, 50], 1, hd, o == "bf16")
    S.check(got, want, tol, o)
  del cache
  torch.cuda.empty_cache()


def test_packed_ignores_rows_outside_the_cache(cuda):
  # arrays that point outside the cache, starts past q's rows: read at the nearest row, nothing outside is touched
  rng = np.random.default_rng(8)
  cache, _ = S.cache(rng, 2, 40, 64, "bf16")
  q = torch.from_numpy(rng.normal(0, 1, (10, 128)).astype(np.float32)).cuda()
  for first, p0, starts in (([1 << 30, -(1 << 30)], [5, 9], [0, 4, 9]), ([0, 0], [1 << 30, -7], [0, 5, 1 << 30]), ([3, 3], [0, 0], [-5, 4, 2])):
    o = torch.zeros(10, 128, device="cuda")
    ops().attention_prefill_packed(q, cache, 2, 1, 64, ints(starts), ints(p0), ints(first), 30, prefix_row=ints([-9]), shared=ints([1 << 30, 2]), o=o)
    torch.cuda.synchronize()
    assert torch.isfinite(o).all()
  o = ops().attention_decode_shared(q, cache, 2, 1, 64, ints([1 << 30] * 10), ints([-(1 << 30)] * 10), ints([1 << 30]), ints([-4] * 5 + [1 << 30] * 5), 20, 10)
  assert torch.isfinite(o).all()


def test_packed_many_sequences(cuda):
  # more sequences than a wave's lanes look through at once, some of them empty, the last round of them not full
  rng = np.random.default_rng(21)
  for n in (64, 65, 150):
    lens = [int(i) for i in rng.integers(0, 9, n)]
    lens[-1], lens[63] = 5, 0
    got, want, tol = packed(22 + n, 2, 1, 64, lens, [int(i) for i in rng.integers(0, 70, n)], 33, pad=3)
    S.check(got, want, tol, n)


def test_many_heads_of_a_key_head(cuda):
  # more query heads a key head than a wave has pairs, and than a workgroup
  for heads in (40, 200):
    got, want, tol = packed(23, heads, 1, 64, [3, 1], [5, 66], 20)
    S.check(got, want, tol, heads)
    got, want, tol = shared(24, heads, 1, 64, 3, 150, 70)
    S.check(got, want, tol, heads)


def test_bounds_past_the_cache(cuda):
  # places and bounds far past the cache: no more keys are read than a prefix and a slot could hold
  rng = np.random.default_rng(25)
  cache, _ = S.cache(rng, 2, 40, 64, "bf16")
  q = torch.from_numpy(rng.normal(0, 1, (6, 128)).astype(np.float32)).cuda()
  o = ops().attention_prefill_packed(q, cache, 2, 1, 64, ints([0, 6]), ints([1 << 30]), ints([0]), 1 << 40)
  assert torch.isfinite(o).all()
  o = ops().attention_decode_shared(q, cache, 2, 1, 64, ints([1 << 30] * 6), ints([3] * 6), ints([0]), ints([1 << 30] * 6), 1 << 40, 1 << 40)
  assert torch.isfinite(o).all()


def test_two_calls_at_once(cuda):
  # the same call on two streams at a time, each with a workspace of its own
  rng = np.random.default_rng(26)
  cache, _ = S.cache(rng, 4, 3000, 64, "bf16")
  q = torch.from_numpy(rng.normal(0, 1, (8, 256)).astype(np.float32)).cuda()
  args = (q, cache, 4, 2, 64, ints([2500] * 8), ints([2600 + 20 * i for i in range(8)]), ints([0]), ints([2490] * 8), 2490, 20)
  want = ops().attention_decode_shared(*args)
  torch.cuda.synchronize()
  streams, outs = [torch.cuda.Stream() for _ in range(2)], []
  for i in range(10):
    with torch.cuda.stream(streams[i % 2]): outs.append(ops().attention_decode_shared(*args))
  torch.cuda.synchronize()
  assert all(torch.equal(o, want) for o in outs)


def shared(seed, heads, kv, hd, batch, prefix, own, fmt="bf16", q="fp32", o="bf16", some=False, tiles=False, max_more=0):
  """A decode call behind a prefix and its oracle: (o, want, tol)."""
  rng = np.random.default_rng(seed)
  sh, mine = np.full(batch, prefix), rng.integers(1, own + 1, batch)
  if some:
    sh = rng.integers(0, prefix + 1, batch)
    sh[0], mine[0] = prefix, 0                  # sees the prefix alone
    if batch > 1: sh[1], mine[1] = 0, 0         # sees nothing
    if batch > 2: sh[2] = 0                     # no prefix
    if batch > 3: mine[3] = -min(3, sh[3])      # its place lies inside the prefix
  first, at = [], prefix + 5
  for m in mine:
    first.append(at)
    at += max(int(m), 0) + int(rng.integers(0, 3))
  cache, values = S.cache(rng, 2 * kv, at + 1, hd, fmt)
  qb = torch.from_numpy(rng.normal(0, 1.5, (batch, heads * hd)).astype(np.float32)).to(S.DTYPE[q])
  out = ops().tiles16(batch, heads * hd) if tiles else None
  got = ops().attention_decode_shared(qb.cuda(), cache, heads, kv, hd, ints(sh + mine - 1), ints(first), ints([2]), ints(sh), prefix + max_more, own + max_more,
                                      o=out, out_dtype=S.DTYPE[o])
  if tiles: got = got.to_rows()
  want, tol = [], []
  for b in range(batch):
    n = int(sh[b] + mine[b])
    w, t = S.attend(qb[b:b + 1], values, S.rows_of(2, int(sh[b]), first[b], max(n, 0)), [n], kv, hd, o == "bf16")
    want.append(w)
    tol.append(t)
  return got, torch.cat(want), torch.cat(tol)


@pytest.mark.parametrize("batch,prefix,own,some", [(1, 1, 1, False), (2, 63, 5, False), (5, 64, 64, True), (4, 65, 1, False), (33, 200, 70, True),
                                                   (7, 1000, 130, True), (3, 0, 90, False), (65, 129, 20, False)])
@pytest.mark.parametrize("heads,kv,hd,fmt,q,o", [(9, 3, 64, "bf16", "fp32", "bf16"), (8, 2, 128, "bfp8", "fp32", "bf16"), (4, 4, 64, "fp32", "fp32", "fp32"),
                                                 (8, 1, 128, "bf16", "bf16", "fp32"), (6, 2, 128, "bfp4", "bf16", "bf16"), (17, 1, 64, "bf16", "fp32", "fp32")])
def test_shared(cuda, batch, prefix, own, some, heads, kv, hd, fmt, q, o):
  print(f"shared {batch} {prefix} {own} {some} {heads}/{kv} {hd} {fmt} {q} {o}", flush=True)
  got, want, tol = shared(11, heads, kv, hd, batch, prefix, own, fmt, q, o, some)
  S.check(got, want, tol, (batch, prefix, fmt))


@pytest.mark.parametrize("fmt", ["bf16", "fp32", "bfp8", "bfp4"])
@pytest.mark.parametrize("hd,heads,kv", [(64, 32, 8), (128, 4, 4)])
@pytest.mark.parametrize("q,o", [("fp32", "fp32"), ("bf16", "bf16"), ("bf16", "fp32")])
def test_shared_types(cuda, fmt, hd, heads, kv, q, o):
  print(f"shared types {fmt} {hd} {heads}/{kv} {q} {o}", flush=True)
  got, want, tol = shared(12, heads, kv, hd, 6, 500, 150, fmt, q, o, True, max_more=700)
  S.check(got, want, tol, (fmt, hd, q, o))


def test_shared_long_prefix_and_tiles(cuda):
  got, want, tol = shared(13, 4, 1, 128, 20, 6000, 300, tiles=True)
  S.check(got, want, tol, "tiles")
  got, want, tol = shared(14, 3, 1, 64, 2, 9001, 1200, fmt="fp32", o="fp32")
  S.check(got, want, tol, "long fp32")


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("fmt,o", [("bf16", "bf16"), ("fp32", "fp32"), ("bf16", "fp32")])
def test_shared_unseen_values(cuda, bad, fmt, o):
  # the prefix's later places and other rows' own keys and values are NaN or infinite: a row that does not see them keeps
  # its result, one that does shows it
  rng = np.random.default_rng(15)
  cache, values = S.cache(rng, 4, 300, 64, fmt)
  q = torch.from_numpy(rng.normal(0, 1, (4, 256)).astype(np.float32))
  sh, first, places = [130, 100, 0, 129], [200, 220, 240, 260], [139, 109, 9, 128]  # (the last sees 129 prefix places alone)
  cache[:, 2 + 129] = bad       # prefix place 129: only row 0 sees it
  cache[:, 210:220] = bad
  cache[:, 250:260] = bad
  cache[:, :2] = bad
  got = ops().attention_decode_shared(q.cuda(), cache, 4, 2, 64, ints(places), ints(first), ints([2]), ints(sh), 130, 40, out_dtype=S.DTYPE[o])
  assert not torch.isfinite(got[0].float()).all()
  for b in (1, 2, 3):
    want, tol = S.attend(q[b:b + 1], values, S.rows_of(2, sh[b], first[b], places[b] + 1), [places[b] + 1], 2, 64, o == "bf16")
    S.check(got[b:b + 1], want, tol, b)


def test_repeats_streams_and_graphs(cuda):
  # the same bits on every call, on another stream, and from two captured graphs that share one workspace and replay in turn
  # with other places in the arrays
  rng = np.random.default_rng(16)
  heads, kv, hd, batch, prefix, own = 8, 2, 128, 9, 700, 60
  cache, _ = S.cache(rng, 2 * kv, prefix + batch * own + 8, hd, "bf16")
  q = torch.from_numpy(rng.normal(0, 1, (batch, heads * hd)).astype(np.float32)).cuda()
  first, prow, sh = ints(prefix + 4 + own * b for b in range(batch)), ints([3]), ints([prefix] * batch)
  spots = [ints(prefix + rng.integers(0, own, batch)) for _ in range(3)]
  starts, p0 = ints([0, 2, 5, 9]), [ints(rng.integers(0, 40, 3)) for _ in range(3)]
  f3, s3 = ints([prefix + 4, prefix + 4 + own, prefix + 4 + 2 * own]), ints([0, 0, 0])
  ws = torch.full((1 << 24,), 255, dtype=torch.uint8, device="cuda")  # (NaN bytes)
  places, places0 = spots[0].clone(), p0[0].clone()
  o1, o2 = torch.zeros_like(q), torch.zeros_like(q)
  dec = lambda p, o: ops().attention_decode_shared(q, cache, heads, kv, hd, p, first, prow, sh, prefix, own, workspace=ws, o=o)
  pre = lambda p, o: ops().attention_prefill_packed(q, cache, heads, kv, hd, starts, p, f3, 800, prefix_row=prow, shared=s3, workspace=ws, o=o)
  eager = [(dec(a, None).clone(), pre(b, None).clone()) for a, b in zip(spots, p0)]
  for a, b, (x, y) in zip(spots, p0, eager): assert torch.equal(dec(a, None), x) and torch.equal(pre(b, None), y)
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side): z = dec(spots[1], None)
  torch.cuda.current_stream().wait_stream(side)
  assert torch.equal(z, eager[1][0])
  torch.cuda.synchronize()
  g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
  with torch.cuda.graph(g1): dec(places, o1)
  with torch.cuda.graph(g2): pre(places0, o2)
  for i in (0, 1, 2, 1, 0):
    places.copy_(spots[i])
    places0.copy_(p0[i])
    o1.fill_(5.0)
    o2.fill_(5.0)
    g1.replay()
    g2.replay()
    assert torch.equal(o1, eager[i][0]) and torch.equal(o2, eager[i][1]), i
    dec(spots[(i + 1) % 3], None)  # (the program's own work in between)
    torch.cuda.synchronize()

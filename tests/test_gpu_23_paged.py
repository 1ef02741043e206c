"""Attention of ragged rows over a cache in pages (fh_attention_paged) against the formula in 64 bits within a bound derived from
each rounding (seq_cases.attend): lengths of none, one and many, pages that end inside a tile, every cache format, pages anywhere,
strides, values that no row may see, captured calls, a workspace shared by two graphs."""
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


def pages_of(rng, counts, spare=2):
  """Each sequence's pages, anywhere in a cache: their tables padded by what no table names, and the cache's pages."""
  ids, at = rng.permutation(sum(counts) + spare), 0
  wide = max(1, max(counts)) + 1
  tables = np.full((len(counts), wide), -7)
  for i, c in enumerate(counts):
    tables[i, :c] = ids[at:at + c]
    tables[i, c:] = [-7, 1 << 30][i % 2]
    at += c
  return tables, len(ids)


def rows_of(table, page, n):
  p = np.arange(max(n, 0))
  return torch.from_numpy(table[p // page] * page + p % page)


def paged(seed, heads, kv, hd, lens, before, page=16, fmt="bf16", q="fp32", o="bf16", ahead=0, pad=0, wide=0, spoil=None, slack=0, apart=0):
  """A call and its oracle: (o, want, tol)."""
  rng = np.random.default_rng(seed)
  n = len(lens)
  tables, count = pages_of(rng, [-(-max(a + b, 0) // page) for a, b in zip(lens, before)])
  cache, values = S.cache(rng, 2 * kv, count * page, hd, fmt)
  T = max(1, ahead + sum(lens) + pad)
  qb = torch.from_numpy(rng.normal(0, 1.5, (T, heads * hd + wide)).astype(np.float32)).to(S.DTYPE[q])
  starts = ahead + np.concatenate([[0], np.cumsum(lens)])
  ob = torch.full((T, heads * hd + wide), 7.0, dtype=S.DTYPE[o], device="cuda")
  if spoil: spoil(cache, tables)
  held = torch.full((n, tables.shape[1] + apart), 1 << 30, dtype=torch.int32, device="cuda")  # (rows further apart than they are wide)
  held[:, :tables.shape[1]] = torch.from_numpy(tables.astype(np.int32)).cuda()
  most = max(1, max(a + b for a, b in zip(lens, before)))
  qg, og = qb.cuda()[:, :heads * hd], ob[:, :heads * hd]
  got = ops().attention_paged(qg, cache, heads, kv, hd, ints(starts), ints(before), held[:, :tables.shape[1]], page, most + slack, o=og)
  assert got.data_ptr() == og.data_ptr()
  want, tol = torch.full((T, heads * hd), 7.0, dtype=torch.float64), torch.zeros(T, heads * hd, dtype=torch.float64)
  for s in range(n):
    a, b, lo = lens[s], before[s], int(starts[s])
    if a: want[lo:lo + a], tol[lo:lo + a] = S.attend(qb[lo:lo + a, :heads * hd], values, rows_of(tables[s], page, a + b), b + 1 + np.arange(a), kv, hd, o == "bf16")
  assert (ob[:, heads * hd:] == 7).all()  # (what lies between o's rows is not o's)
  return got, want, tol


@pytest.mark.parametrize("lens,before,page", [
  ([1], [0], 16), ([1], [15], 16), ([1], [16], 16), ([1, 1, 1, 1], [63, 64, 65, 700], 16), ([1] * 9, [5, 90, 0, 1000, 3, 128, 127, 129, 64], 64),
  ([20, 1, 30], [0, 40, 0], 32), ([64, 0, 63, 65], [0, 5, 1, 64], 16), ([129, 32, 1, 33], [0, 100, 517, 0], 128), ([260, 1], [7, 2000], 16),
  ([0, 0, 3, 0], [4, 0, 0, 9], 64), ([2, 5, 8, 4], [300, 40, 0, 1111], 16), ([1, 1, 2], [-1, 10, -1], 32)])
@pytest.mark.parametrize("heads,kv,hd,fmt,q,o", [(9, 3, 64, "bf16", "fp32", "bf16"), (8, 2, 128, "bfp8", "fp32", "bf16"), (4, 4, 64, "fp32", "fp32", "fp32"),
                                                 (8, 1, 128, "bf16", "bf16", "fp32"), (6, 2, 128, "bfp4", "bf16", "bf16"), (5, 1, 64, "bf16", "fp32", "fp32")])
def test_paged(cuda, lens, before, page, heads, kv, hd, fmt, q, o):
  print(f"paged {lens} {before} {page} {heads}/{kv} {hd} {fmt} {q} {o}", flush=True)
  got, want, tol = paged(1, heads, kv, hd, lens, before, page, fmt, q, o)
  S.check(got, want, tol, (lens, fmt))


@pytest.mark.parametrize("fmt", ["bf16", "fp32", "bfp8", "bfp4"])
@pytest.mark.parametrize("hd,heads,kv", [(64, 16, 1), (128, 5, 5), (128, 32, 1)])
@pytest.mark.parametrize("q,o", [("fp32", "fp32"), ("bf16", "bf16"), ("fp32", "bf16"), ("bf16", "fp32")])
def test_paged_types(cuda, fmt, hd, heads, kv, q, o):
  print(f"paged types {fmt} {hd} {heads}/{kv} {q} {o}", flush=True)
  for lens, before in (([70, 3, 11], [9, 40, 120]), ([1, 1, 1], [200, 17, 90])):
    got, want, tol = paged(2, heads, kv, hd, lens, before, 16, fmt, q, o)
    S.check(got, want, tol, (fmt, hd, q, o))


def test_strides_and_rows_behind(cuda):
  # rows before the first start and behind the last sequence keep what they held; q, o and tables are columns of wider buffers
  for lens, before in (([40, 0, 25], [0, 0, 3]), ([1, 1, 1, 0, 1], [100, 0, 333, 5, 64])):
    got, want, tol = paged(3, 6, 2, 64, lens, before, ahead=5, pad=13, wide=24, apart=3)
    S.check(got, want, tol, "strides")
    assert (got[:5] == 7).all() and (got[5 + sum(lens):] == 7).all()


@pytest.mark.parametrize("heads,kv,hd,fmt,q,o", [(64, 64, 128, "bf16", "bf16", "bf16"), (80, 80, 64, "bf16", "fp32", "fp32"), (64, 64, 128, "bfp8", "fp32", "bf16"),
                                                 (80, 80, 64, "bfp4", "bf16", "fp32")])
def test_many_tiles(cuda, heads, kv, hd, fmt, q, o):
  # more tiles of prompts than workgroups that the GPU holds: a tile a workgroup, with sequences of none and one among them
  lens, before = [300, 1, 0, 129, 128, 142], [0, 30, 5, 0, 17, 0]
  got, want, tol = paged(20, heads, kv, hd, lens, before, 16, fmt, q, o, ahead=3, pad=9)
  S.check(got, want, tol, (heads, hd, fmt))
  assert (got[:3] == 7).all() and (got[3 + sum(lens):] == 7).all()


def test_long_contexts(cuda):
  # few rows after many (the keys' long axis), with the bound of the context far above what is there
  got, want, tol = paged(4, 8, 2, 128, [3, 40], [2000, 1111], 64, slack=3000)
  S.check(got, want, tol, "long")
  got, want, tol = paged(5, 3, 1, 64, [1, 2], [1500, 700], 16, fmt="fp32", o="fp32")
  S.check(got, want, tol, "long fp32")
  got, want, tol = paged(6, 4, 1, 128, [1] * 5, [9000, 3, 0, 4097, 640], 16)
  S.check(got, want, tol, "long tokens")


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("fmt,o", [("bf16", "bf16"), ("fp32", "fp32"), ("bf16", "fp32")])
def test_unseen_values(cuda, bad, fmt, o):
  # pages of nobody, a later token's place and the rest of a sequence's last page are NaN or infinite: rows that do not see
  # them keep their results; a row that sees one is not finite
  cut = 37  # (the first sequence's place 37: its rows 0 .. 36 do not see it)
  def spoil(cache, tables):
    used = np.concatenate([rows_of(tables[0], 16, 90), rows_of(tables[1], 16, 24), rows_of(tables[2], 16, 71)])
    rest = np.setdiff1d(np.arange(cache.shape[1]), used)
    cache[:, torch.from_numpy(rest)] = bad
    cache[:, int(rows_of(tables[0], 16, 90)[cut])] = bad
  got, want, tol = paged(7, 4, 2, 64, [90, 20, 1], [0, 4, 70], 16, fmt, "fp32", o, spoil=spoil)
  S.check(got[:cut], want[:cut], tol[:cut], "before the place")
  S.check(got[90:], want[90:], tol[90:], "the other sequences")
  assert not torch.isfinite(got[cut:90].float()).all(1).any()
  # the same for single tokens alone
  def one(cache, tables):
    used = np.concatenate([rows_of(tables[i], 16, c) for i, c in enumerate((90, 24, 300))])
    cache[:, torch.from_numpy(np.setdiff1d(np.arange(cache.shape[1]), used))] = bad
    cache[:, int(rows_of(tables[1], 16, 24)[11])] = bad
  got, want, tol = paged(8, 4, 2, 64, [1, 1, 1], [89, 23, 299], 16, fmt, "fp32", o, spoil=one)
  S.check(got[[0, 2]], want[[0, 2]], tol[[0, 2]], "the other tokens")
  assert not torch.isfinite(got[1].float()).all()


def test_past_32_bits(cuda):
  # a cache whose values lie past 2^31 elements: the last pages of the last plane
  rows, hd = 17 << 20, 64
  cache = torch.zeros(2, rows, hd, dtype=torch.bfloat16, device="cuda")
  rng = np.random.default_rng(9)
  some = torch.from_numpy(rng.normal(0, 1, (2, 64, hd)).astype(np.float32)).to(torch.bfloat16)
  cache[:, rows - 64:] = some.cuda()
  tables = ints([rows // 16 - 1, rows // 16 - 3, rows // 16 - 4, rows // 16 - 2]).view(1, 4)
  values = some.double().view(2, 4, 16, hd)[:, [3, 1, 0, 2]].reshape(2, 64, hd)
  for n, p0 in ((30, 20), (1, 49)):
    q = torch.from_numpy(rng.normal(0, 1, (n, 2 * hd)).astype(np.float32))
    got = ops().attention_paged(q.cuda(), cache, 2, 1, hd, ints([0, n]), ints([p0]), tables, 16, 64, out_dtype=torch.bfloat16)
    want, tol = S.attend(q, values, torch.arange(64), p0 + 1 + np.arange(n), 1, hd, True)
    S.check(got, want, tol, n)


def test_pages_and_places_outside(cuda):
  # tables, places, starts and bounds that point anywhere: read at the nearest page, nothing outside touched
  rng = np.random.default_rng(10)
  cache, _ = S.cache(rng, 2, 48, 64, "bf16")
  q = torch.from_numpy(rng.normal(0, 1, (10, 128)).astype(np.float32)).cuda()
  for starts, p0, tables, bound in (([0, 5, 10], [100, 3], [[1 << 30, -5], [2, 9]], 30), ([-3, 2, 40], [0, -20], [[0, 1], [7, 7]], 1 << 40),
                                    ([0, 10, 4], [1 << 30, 5], [[-(1 << 31), 2], [1, 1]], 1 << 40), ([0, 1, 2], [1 << 30, 31], [[3, -1], [0, 2]], 32)):
    o = torch.zeros(10, 128, device="cuda")
    ops().attention_paged(q, cache, 2, 1, 64, ints(starts), ints(p0), torch.tensor(tables, dtype=torch.int32, device="cuda"), 16, bound, o=o)
    torch.cuda.synchronize()
    assert torch.isfinite(o).all()


def test_many_sequences_and_heads(cuda):
  # more sequences than a wave's lanes look through at once, some empty; more heads a key head than a workgroup has pairs
  rng = np.random.default_rng(11)
  for n in (64, 65, 150):
    for single in (True, False):
      lens = [int(i) for i in (rng.integers(0, 2, n) if single else rng.integers(0, 9, n))]
      lens[-1], lens[63] = 1 if single else 5, 0
      got, want, tol = paged(12 + n, 2, 1, 64, lens, [int(i) for i in rng.integers(0, 170, n)], 16, pad=3)
      S.check(got, want, tol, n)
  for heads in (40, 200):
    for lens in ([3, 1], [1, 1]):
      got, want, tol = paged(13, heads, 1, 64, lens, [5, 166], 32)
      S.check(got, want, tol, heads)


def test_as_the_packed_attention(cuda):
  # pages in order are a cache of slots: the packed prompts' values, within both bounds
  rng = np.random.default_rng(14)
  cache, _ = S.cache(rng, 4, 640, 64, "bf16")
  q = torch.from_numpy(rng.normal(0, 1, (60, 4 * 64)).astype(np.float32)).cuda()
  starts, p0, first = ints([0, 20, 21, 60]), ints([30, 150, 0]), ints([0, 160, 320])
  a = ops().attention_prefill_packed(q, cache, 4, 2, 64, starts, p0, first, 151)
  b = ops().attention_paged(q, cache, 4, 2, 64, starts, p0, torch.arange(30, dtype=torch.int32, device="cuda").view(3, 10), 16, 151)
  assert float((a - b).abs().max()) <= 2.0 ** -18 * float(a.abs().max()) * 4


def test_repeats_streams_and_graphs(cuda):
  # the same bits on every call, on another stream, and from two captured graphs that share one workspace and replay in turn
  # with other tables and places in the arrays
  rng = np.random.default_rng(15)
  heads, kv, hd, n = 8, 2, 128, 9
  cache, _ = S.cache(rng, 2 * kv, 16 * 400, hd, "bf16")
  q = torch.from_numpy(rng.normal(0, 1, (40, heads * hd)).astype(np.float32)).cuda()
  one, many = ints(range(n + 1)), ints([0, 2, 5, 5, 6, 20, 21, 22, 39, 40])
  spots = [ints(rng.integers(0, 600, n)) for _ in range(3)]
  tabs = [torch.from_numpy(rng.permutation(400)[:n * 40].reshape(n, 40).astype(np.int32)).cuda() for _ in range(3)]
  ws = ops().attention_paged_workspace(40, n, heads, kv, hd, 640).fill_(255)  # (NaN bytes)
  dec = lambda p, t, o: ops().attention_paged(q[:n], cache, heads, kv, hd, one, p, t, 16, 640, workspace=ws, o=o)
  pre = lambda p, t, o: ops().attention_paged(q, cache, heads, kv, hd, many, p, t, 16, 640, workspace=ws, o=o)
  eager = [(dec(a, t, None).clone(), pre(a, t, None).clone()) for a, t in zip(spots, tabs)]
  for a, t, (x, y) in zip(spots, tabs, eager): assert torch.equal(dec(a, t, None), x) and torch.equal(pre(a, t, None), y)
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side): z = dec(spots[1], tabs[1], None)
  torch.cuda.current_stream().wait_stream(side)
  assert torch.equal(z, eager[1][0])
  torch.cuda.synchronize()
  places, table = spots[0].clone(), tabs[0].clone()
  o1, o2 = torch.zeros(n, heads * hd, device="cuda"), torch.zeros(40, heads * hd, device="cuda")
  g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
  with torch.cuda.graph(g1): dec(places, table, o1)
  with torch.cuda.graph(g2): pre(places, table, o2)
  for i in (0, 1, 2, 1, 0):
    places.copy_(spots[i])
    table.copy_(tabs[i])
    o1.fill_(5.0)
    o2.fill_(5.0)
    g1.replay()
    g2.replay()
    assert torch.equal(o1, eager[i][0]) and torch.equal(o2, eager[i][1]), i
    dec(spots[(i + 1) % 3], tabs[i], None)  # (the program's own work in between)
    torch.cuda.synchronize()


def test_two_calls_at_once(cuda):
  # the same call on two streams at a time, each with a workspace of its own
  rng = np.random.default_rng(16)
  cache, _ = S.cache(rng, 4, 3200, 64, "bf16")
  q = torch.from_numpy(rng.normal(0, 1, (8, 256)).astype(np.float32)).cuda()
  tables = torch.from_numpy(rng.integers(0, 200, (8, 190)).astype(np.int32)).cuda()
  args = (q, cache, 4, 2, 64, ints(range(9)), ints(rng.integers(0, 3000, 8)), tables, 16, 3000)
  want = ops().attention_paged(*args)
  torch.cuda.synchronize()
  streams, outs = [torch.cuda.Stream() for _ in range(2)], []
  for i in range(10):
    with torch.cuda.stream(streams[i % 2]): outs.append(ops().attention_paged(*args))
  torch.cuda.synchronize()
  assert all(torch.equal(o, want) for o in outs)


def test_a_workspace_for_more_serves_less(cuda):
  rng = np.random.default_rng(17)
  cache, _ = S.cache(rng, 4, 3200, 128, "bf16")
  ws = ops().attention_paged_workspace(50, 8, 8, 2, 128, 3000)
  ws.fill_(255)
  q = torch.from_numpy(rng.normal(0, 1, (50, 1024)).astype(np.float32)).cuda()
  tables = torch.from_numpy(rng.integers(0, 200, (8, 190)).astype(np.int32)).cuda()
  for n, heads, bound in ((1, 8, 3000), (8, 2, 100), (8, 8, 2999), (3, 4, 65)):
    for step in (1, 6):
      a = (q[:n * step, :heads * 128], cache, heads, 2, 128, ints(step * i for i in range(n + 1)), ints(rng.integers(0, bound, n)), tables[:n], 16, bound)
      assert torch.equal(ops().attention_paged(*a, workspace=ws), ops().attention_paged(*a)), (n, heads, bound, step)

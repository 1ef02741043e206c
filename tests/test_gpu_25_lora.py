"""Each row's low-rank adapter beside a shared projection (fh_lora) against the formula in 64 bits. Errors are bounded by the roundings
(eps = 2^-24): u = x A^T is a sum of K products, each of x's and A's terms (off by at most c of themselves: 4 2^-16 for bf16 output, whose
fp32 values go in as two bf16 terms, 8 2^-24 for fp32 output, three), and the sum itself by K + 40 eps of sum |x A|; u B^T the same with
rank; then the addition, and the output's rounding, half a step."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPE = {"fp32": torch.float32, "bf16": torch.bfloat16}


def ops():
  from ferrite_amd import ops as m
  return m


def ints(v):
  return torch.tensor(list(v), dtype=torch.int32, device="cuda")


def made(seed, n, K, parts, rank, w="bf16", scaled=True):
  rng = np.random.default_rng(seed)
  N, S = sum(parts), len(parts)
  a = torch.from_numpy(rng.normal(0, K ** -0.5, (n, S * rank, K)).astype(np.float32)).to(DTYPE[w])
  b = torch.from_numpy(rng.normal(0, 0.5, (n, N, rank)).astype(np.float32)).to(DTYPE[w])
  s = torch.from_numpy(rng.normal(1, 0.3, n).astype(np.float32)) if scaled else None
  return ops().Adapters(a.cuda(), b.cuda(), None if s is None else s.cuda(), tuple(parts))


def formula(x, ad, ids, residual, y_bf16):
  """The result in 64 bits, and the bound."""
  eps, c = 2.0 ** -24, 4 * 2.0 ** -16 if y_bf16 else 8 * 2.0 ** -24
  a, b, s = ad.a.double().cpu(), ad.b.double().cpu(), None if ad.scale is None else ad.scale.double().cpu()
  n, C, K = a.shape
  r, T, N = b.shape[2], x.shape[0], b.shape[1]
  x = x.double().cpu()
  y = torch.zeros(T, N, dtype=torch.float64) if residual is None else residual.double().cpu().clone()
  tol, base = torch.zeros_like(y), y.abs()
  for i in range(n):
    rows = [t for t, v in enumerate(ids) if v == i]
    if not rows: continue
    u, size = x[rows] @ a[i].T, x[rows].abs() @ a[i].abs().T
    eu, at, f = (c + (K + 40) * eps) * size, 0, 1.0 if s is None else float(s[i])
    for p, cols in enumerate(ad.parts):
      us, B = u[:, p * r:(p + 1) * r], b[i, at:at + cols]
      y[rows, at:at + cols] += f * (us @ B.T)
      tol[rows, at:at + cols] = abs(f) * (eu[:, p * r:(p + 1) * r] @ B.abs().T + (c + (r + 40) * eps) * (us.abs() @ B.abs().T))
      at += cols
    tol[rows] += 2 * eps * (base[rows] + y[rows].abs())
  if y_bf16: tol = tol + 2.0 ** -8 * (y.abs() + tol) * torch.tensor([[v in range(n)] for v in ids])
  return y, tol


def run(seed, ids, K, parts, rank, n, x="bf16", w="bf16", y="fp32", wide=0, in_place=False, plain=False, scaled=True):
  rng = np.random.default_rng(seed)
  T, N = len(ids), sum(parts)
  ad = made(seed, n, K, parts, rank, w, scaled)
  xb = torch.from_numpy(rng.normal(0, 1, (T, K + wide)).astype(np.float32)).to(DTYPE[x]).cuda()
  base = torch.from_numpy(rng.normal(0, 1, (T, N + wide)).astype(np.float32)).to(DTYPE[y]).cuda()
  xs, res = xb[:, :K], None if plain else base[:, :N]
  want, tol = formula(xs, ad, ids, res, y == "bf16")
  out = res if in_place else torch.full((T, N + wide), 7.0, dtype=DTYPE[y], device="cuda")[:, :N]
  behind = base[:, N:].clone()
  got = ops().lora(xs, ad, ints(ids), residual=res, out=out)
  assert got.data_ptr() == out.data_ptr() and torch.equal(base[:, N:], behind)
  bad = (got.double().cpu() - want).abs() > tol
  assert torch.isfinite(got.float()).all() and not bad.any(), (int(bad.sum()), float(((got.double().cpu() - want).abs() / tol.clamp(min=1e-30)).max()))
  return got


TOKENS = {"one": [0], "none": [-1], "two": [1, 1], "mixed": [2, -1, 0, 2, 5, 1, 1, -3, 0], "each": list(range(17)), "past": [99, 3, 1 << 30, -(1 << 31), 3]}


@pytest.mark.parametrize("ids", list(TOKENS))
@pytest.mark.parametrize("K,parts,rank", [(576, (576, 192, 192), 8), (512, (256,), 16), (1000, (24, 8), 40), (72, (8, 64, 16, 40), 24), (4096, (128, 128), 64), (8, (8,), 128)])
@pytest.mark.parametrize("x,w,y", [("bf16", "bf16", "fp32"), ("fp32", "bf16", "bf16"), ("fp32", "fp32", "fp32")])
def test_tokens(cuda, ids, K, parts, rank, x, w, y):
  print(f"lora tokens {ids} {K} {parts} {rank} {x} {w} {y}", flush=True)
  run(1, TOKENS[ids], K, parts, rank, 17, x, w, y)


@pytest.mark.parametrize("x", ["fp32", "bf16"])
@pytest.mark.parametrize("w", ["fp32", "bf16"])
@pytest.mark.parametrize("y", ["fp32", "bf16"])
def test_types(cuda, x, w, y):
  print(f"lora types {x} {w} {y}", flush=True)
  ids = [0] * 70 + [-1] * 9 + [2] * 33 + [1, 0, 1, 0, -1, 2] * 6
  for rank in (8, 48):
    run(2, ids, 328, (272, 96), rank, 3, x, w, y)
    run(3, ids, 328, (272, 96), rank, 3, x, w, y, in_place=True, scaled=False)
    run(4, ids, 328, (272, 96), rank, 3, x, w, y, plain=True)


@pytest.mark.parametrize("rows", [15, 16, 17, 63, 64, 65, 130, 1025, 1100])
def test_rows(cuda, rows):
  # tiles of rows that end inside, of one adapter, of few and of many, and past the rows up to which a tile's adapters are shared out
  rng = np.random.default_rng(rows)
  print(f"lora rows {rows}", flush=True)
  for ids in ([0] * rows, [int(i) for i in np.sort(rng.integers(-1, 5, rows))], [int(i) for i in rng.integers(-1, 70, rows)]):
    run(5, ids, 200, (80, 48), 16, 70)


def test_strides(cuda):
  # x, residual and out are columns of wider buffers
  run(6, [0, 1, -1, 1] * 20, 256, (64, 32), 8, 2, wide=24)
  run(7, [0, 1, -1, 1] * 20, 256, (64, 32), 8, 2, "fp32", "bf16", "bf16", wide=8, in_place=True)


def test_rows_with_no_adapter_keep_their_bits(cuda):
  got = torch.randn(70, 64, device="cuda")
  want = got.clone()
  ad = made(8, 3, 64, (64,), 8)
  x = torch.full((70, 64), float("nan"), device="cuda")
  x[5] = 1.0
  ids = ints([-1] * 5 + [2] + [3] * 64)
  ops().lora(x, ad, ids, residual=got, out=got)
  keep = [t for t in range(70) if t != 5]
  assert torch.equal(got[keep], want[keep]) and torch.isfinite(got).all() and not torch.equal(got[5], want[5])
  out = ops().lora(x, ad, ids)
  assert (out[keep] == 0).all() and torch.equal(out[5], out[5]) and (out[5] != 0).any()
  # one row's values that are not finite stay that row's
  x = torch.randn(70, 64, device="cuda")
  clean = ops().lora(x, ad, ints([1] * 70))
  x[9], x[40, 3] = float("nan"), float("inf")
  spoilt = ops().lora(x, ad, ints([1] * 70))
  rest = [t for t in range(70) if t not in (9, 40)]
  assert torch.equal(clean[rest], spoilt[rest]) and not torch.isfinite(spoilt[9]).any() and not torch.isfinite(spoilt[40]).any()


def test_wide_and_long(cuda):
  # y past 2^31 elements: its last rows (the ones before have no adapter)
  T, N = 70000, 32768
  y = torch.zeros(T, N, dtype=torch.bfloat16, device="cuda")
  ad = made(9, 2, 64, (N,), 8, scaled=False)
  x = torch.zeros(T, 64, dtype=torch.bfloat16, device="cuda")
  x[-3:] = torch.randn(3, 64, device="cuda").to(torch.bfloat16)
  ids = torch.full((T,), -1, dtype=torch.int32, device="cuda")
  ids[-3:] = 1
  ops().lora(x, ad, ids, residual=y, out=y)
  want, tol = formula(x[-3:], ad, [1, 1, 1], torch.zeros(3, N), True)
  assert ((y[-3:].double().cpu() - want).abs() <= tol).all() and float(y[:-3].abs().max()) == 0


def test_repeats_streams_and_graphs(cuda):
  # the same bits on every call and stream, and from two graphs that share a workspace of NaN bytes and replay with other ids
  rng = np.random.default_rng(10)
  ad, x = made(10, 6, 512, (128, 64), 16), torch.randn(90, 512, device="cuda")
  base = torch.randn(90, 192, device="cuda")
  sets = [ints(rng.integers(-1, 6, 90)) for _ in range(3)]
  ws = ops().lora_workspace(200, ad)
  ws.fill_(255)
  call = lambda n, ids, out: ops().lora(x[:n], ad, ids[:n], residual=base[:n], out=out, workspace=ws)
  eager = [(call(90, i, None).clone(), call(7, i, None).clone()) for i in sets]
  for i, (a, b) in zip(sets, eager): assert torch.equal(call(90, i, None), a) and torch.equal(call(7, i, None), b)
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side): z = call(90, sets[1], None)
  torch.cuda.current_stream().wait_stream(side)
  assert torch.equal(z, eager[1][0])
  torch.cuda.synchronize()
  ids, o1, o2 = sets[0].clone(), torch.zeros(90, 192, device="cuda"), torch.zeros(7, 192, device="cuda")
  g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
  with torch.cuda.graph(g1): call(90, ids, o1)
  with torch.cuda.graph(g2): call(7, ids, o2)
  for i in (0, 1, 2, 1, 0):
    ids.copy_(sets[i])
    o1.fill_(5.0)
    o2.fill_(5.0)
    g1.replay()
    g2.replay()
    assert torch.equal(o1, eager[i][0]) and torch.equal(o2, eager[i][1]), i
    call(90, sets[(i + 1) % 3], None)
    torch.cuda.synchronize()


def test_pack_adapters(cuda):
  # ranks that differ, a part left alone, from a checkpoint's matrices
  rng = np.random.default_rng(11)
  m = lambda *s: torch.from_numpy(rng.normal(0, 0.3, s).astype(np.float32)).to(torch.bfloat16)
  given = [[(m(4, 96), m(32, 4)), None], [(m(11, 96), m(32, 11)), (m(1, 96), m(16, 1))], [None, (m(16, 96), m(16, 16))]]
  ad = ops().pack_adapters(given, (32, 16), scales=[2.0, 0.5, 1.0])
  assert ad.rank == 16 and ad.a.shape == (3, 32, 96) and ad.b.shape == (3, 48, 16)
  x, ids = m(9, 96), [0, 1, 2, 2, 1, 0, -1, 1, 0]
  got = ops().lora(x.cuda(), ad, ints(ids)).double().cpu()
  want, tol = torch.zeros(9, 48, dtype=torch.float64), formula(x, ad, ids, None, False)[1]
  for t, i in enumerate(ids):
    for (lo, hi), ab in zip(((0, 32), (32, 48)), given[i] if i >= 0 else (None, None)):
      if ab is not None: want[t, lo:hi] = [2.0, 0.5, 1.0][i] * ((x[t].double() @ ab[0].double().T) @ ab[1].double().T)
  assert ((got - want).abs() <= tol).all()
  with pytest.raises(ValueError): ops().pack_adapters([[(m(4, 96), m(32, 4))]], (32, 16))
  with pytest.raises(ValueError): ops().pack_adapters([[(m(4, 96), m(30, 4)), None]], (32, 16))


@pytest.mark.parametrize("x,o", [("fp32", "bf16"), ("bf16", "fp32"), ("fp32", "fp32"), ("bf16", "bf16")])
@pytest.mark.parametrize("T,split", [(1, 8), (3, 1544), (70, 264)])
def test_silu_gate_rows(cuda, T, split, x, o):
  # expf within 2 units (2^-22 of it), its sum, the quotient and the product a rounding each (2^-24), o's own: 2^-21 with room
  dt = dict(fp32=torch.float32, bf16=torch.bfloat16)
  buf = (torch.randn(T, 2 * split + 16, device="cuda") * 8).to(dt[x])
  out = torch.full((T, split + 8), 7.0, dtype=dt[o], device="cuda")
  buf[0, 0], buf[0, split] = -200., 3.  # (a gate whose exponential overflows: 0)
  got = ops().silu_gate_rows(buf[:, :2 * split], split, out[:, :split])
  g, u = buf[:, :split].double().cpu(), buf[:, split:2 * split].double().cpu()
  want = g * torch.sigmoid(g) * u
  tol = want.abs() * (2.0 ** -21 + torch.finfo(dt[o]).eps / 2) + 2.0 ** -126
  assert ((got.double().cpu() - want).abs() <= tol).all() and (out[:, split:] == 7).all()

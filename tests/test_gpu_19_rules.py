"""Logit rules (fh_logit_rules) against the formula in 64 bits: penalties by a row's tokens and their counts, biases (an id
given twice too), grammar masks (one that leaves nothing too), padding, odd widths and strides, in place, captured."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def ops():
  from ferrite_amd import ops as m
  return m


def oracle(x, tokens=None, lengths=None, prompts=None, rep=None, pre=None, fre=None, ids=None, bias=None, allowed=None):
  """The rules in 64 bits, and a bound of the error: a rounding (2^-24) of each step's value and of the terms added."""
  R, V = x.shape
  y = x.astype(np.float64)
  size = np.abs(y)
  for r in range(R):
    if tokens is not None:
      n = tokens.shape[1] if lengths is None else max(0, min(int(lengths[r]), tokens.shape[1]))
      t = tokens[r, :n].astype(np.int64)
      after = t[max(0, 0 if prompts is None else int(prompts[r])):]
      seen = np.unique(t[(t >= 0) & (t < V)])
      k = 1.0 if rep is None else float(rep[r])
      y[r, seen] = np.where(y[r, seen] > 0, y[r, seen] / k, y[r, seen] * k)
      size[r, seen] = np.maximum(size[r, seen], np.abs(y[r, seen]))
      count = np.bincount(after[(after >= 0) & (after < V)], minlength=V)
      less = (0.0 if fre is None else float(fre[r])) * count + (0.0 if pre is None else float(pre[r])) * (count > 0)
      y[r] -= less
      size[r] += np.abs(less)
    if ids is not None:
      for i, b in zip(ids[r], bias[r]):
        if 0 <= i < V:
          y[r, i] += float(b)
          size[r, i] += abs(float(b))
  if allowed is not None:
    bits = (allowed.view(np.uint32)[:, np.arange(V) // 32] >> (np.arange(V) % 32).astype(np.uint32)) & 1
    y = np.where(bits > 0, y, -np.inf)
  # (at most 8 roundings of values no larger than `size`, and the sum of a column's biases: one a term)
  return y, (8 + (0 if ids is None else ids.shape[1])) * 2.0 ** -24 * size


def check(got, want, tol):
  got = got.cpu().numpy().astype(np.float64)
  fine = np.isfinite(want)
  assert np.array_equal(got[~fine], want[~fine], equal_nan=True)
  assert (np.abs(got[fine] - want[fine]) <= tol[fine]).all(), float((np.abs(got[fine] - want[fine]) / np.maximum(tol[fine], 1e-30)).max())


def case(seed, R, V, H=0, nb=0, mask=False, scalars=True):
  rng = np.random.default_rng(seed)
  x = rng.normal(0, 3, (R, V)).astype(np.float32)
  c = dict(tokens=None, lengths=None, prompts=None, rep=None, pre=None, fre=None, ids=None, bias=None, allowed=None)
  if H:
    t = rng.integers(0, V, (R, H)).astype(np.int32)
    t[:, ::2] = rng.integers(0, min(V, 9), t[:, ::2].shape)   # a few columns many times
    t[:, 1::7] = -1                                            # padding
    t[:, 2::11] = V + rng.integers(0, 5)                       # outside the vocabulary
    c.update(tokens=t, lengths=rng.integers(0, H + 1, R).astype(np.int32), prompts=rng.integers(0, H + 1, R).astype(np.int32))
    c["lengths"][0] = H
  if scalars:
    c.update(rep=rng.uniform(0.8, 1.5, R).astype(np.float32), pre=rng.uniform(-1, 1, R).astype(np.float32), fre=rng.uniform(-0.2, 0.3, R).astype(np.float32))
  if nb:
    c.update(ids=rng.integers(-1, V + 1, (R, nb)).astype(np.int32), bias=rng.normal(0, 4, (R, nb)).astype(np.float32))
    c["ids"][:, nb // 2:] = c["ids"][:, :nb - nb // 2]         # every id twice
  if mask:
    c["allowed"] = rng.integers(-(1 << 31), 1 << 31, (R, -(-V // 32))).astype(np.int32)
    c["allowed"][0] = 0                                        # a row with nothing left
  return x, c


def run(x, c, **kw):
  g = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()
  return ops().logit_rules(x if isinstance(x, torch.Tensor) else g(x), tokens=g(c["tokens"]), lengths=g(c["lengths"]), prompt_lengths=g(c["prompts"]), repetition=g(c["rep"]),
                           presence=g(c["pre"]), frequency=g(c["fre"]), bias_ids=g(c["ids"]), bias=g(c["bias"]), allowed=g(c["allowed"]), **kw)


@pytest.mark.parametrize("R,V,H,nb,mask", [(1, 1, 3, 1, True), (1, 31, 10, 0, True), (3, 33, 0, 5, True), (2, 1000, 300, 0, False), (5, 4096, 77, 40, True),
                                           (4, 4097, 1, 2, True), (2, 50257, 3000, 300, True), (1, 128256, 20000, 0, False), (9, 128256, 500, 1024, True),
                                           (130, 2049, 64, 3, True), (3, 262144, 9, 0, True), (2, 70001, 0, 0, True), (2, 257, 0, 0, False)])
def test_rules(cuda, R, V, H, nb, mask):
  print(f"rules {R} x {V}, history {H}, {nb} biases, mask {mask}", flush=True)
  x, c = case(R + V, R, V, H, nb, mask)
  check(run(x, c), *oracle(x, **c))


def test_each_argument_alone(cuda):
  x, c = case(3, 3, 5000, 200, 20, True)
  none = dict.fromkeys(c)
  groups = [("tokens",), ("tokens", "lengths", "rep"), ("tokens", "prompts", "pre"), ("tokens", "fre"), ("ids", "bias"), ("allowed",), ("rep", "pre", "fre"), ()]
  for names in groups:
    some = {**none, **{n: c[n] for n in names}}
    check(run(x, some), *oracle(x, **some))


def test_infinite_logits_and_values_under_the_mask(cuda):
  # NaN and infinities where the mask is 0 become -inf; unmasked ones stay what the formula makes of them
  x, c = case(4, 2, 3000, 100, 0, True)
  x[1, ::3], x[1, 1::3] = np.nan, np.inf
  x[1, 2::9] = -np.inf
  c["allowed"][1] = 0x55555555
  got = run(x, c).cpu().numpy()
  bits = np.arange(3000) % 2 == 0
  assert (got[0] == -np.inf).all() and (got[1, ~bits] == -np.inf).all()
  assert np.array_equal(np.isnan(got[1, bits]), np.isnan(x[1, bits])) and (got[1, bits & (np.arange(3000) % 3 == 1)] == np.inf).all()


def test_strides_in_place_and_broadcast(cuda):
  # columns of a wider buffer whose rows are not 16-byte aligned; in place; one row's mask expanded to all rows
  x, c = case(5, 6, 1003, 50, 7, True)
  c["allowed"][0] = c["allowed"][1]
  wide = torch.full((6, 1100), 9.0, device="cuda")
  view = wide[:, 3:1006]
  view.copy_(torch.from_numpy(x))
  want, tol = oracle(x, **c)
  check(run(view, c), want, tol)
  got = run(view, c, out=view)
  assert got.data_ptr() == view.data_ptr()
  check(view, want, tol)
  assert (wide[:, :3] == 9).all() and (wide[:, 1006:] == 9).all()
  one = torch.from_numpy(c["allowed"][1:2].copy()).cuda().expand(6, -1)
  got = ops().logit_rules(torch.from_numpy(x).cuda(), allowed=one)
  want, tol = oracle(x, allowed=np.repeat(c["allowed"][1:2], 6, 0))
  check(got, want, tol)


def test_repeats_and_graph(cuda):
  # the same bits every time (biases of one id added in their order), and from a graph whose arrays change between replays
  x, c = case(6, 4, 20000, 900, 600, True)
  c["ids"][:] = c["ids"][:, :1] % 20000  # (one column, 600 times)
  first = run(x, c)
  check(first, *oracle(x, **c))
  for _ in range(3): assert torch.equal(run(x, c), first)
  cases = [case(s, 4, 20000, 900, 60, True) for s in (7, 8, 9)]
  dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
  eager = [run(a, b) for a, b in cases]
  X = dev(cases[0][0])
  held = {k: dev(v) for k, v in cases[0][1].items()}
  names = dict(tokens="tokens", lengths="lengths", prompt_lengths="prompts", repetition="rep", presence="pre", frequency="fre", bias_ids="ids", bias="bias", allowed="allowed")
  out = torch.empty_like(X)
  torch.cuda.synchronize()
  g = torch.cuda.CUDAGraph()
  with torch.cuda.graph(g): ops().logit_rules(X, out=out, **{a: held[b] for a, b in names.items()})
  for i in (0, 1, 2, 1, 0):
    X.copy_(dev(cases[i][0]))
    for k, v in cases[i][1].items(): held[k].copy_(dev(v))
    g.replay()
    assert torch.equal(out, eager[i]), i
    run(*cases[(i + 1) % 3])
    torch.cuda.synchronize()


def test_large_batch_captured(cuda):
  # the widest parts (more LDS than a launch has unasked), from a graph, against the eager call
  x, c = case(10, 128, 128256, 40, 1024, False)
  dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
  X, held = dev(x), {k: dev(v) for k, v in c.items() if v is not None}
  args = dict(tokens=held["tokens"], lengths=held["lengths"], prompt_lengths=held["prompts"], repetition=held["rep"], presence=held["pre"],
              frequency=held["fre"], bias_ids=held["ids"], bias=held["bias"])
  eager = ops().logit_rules(X, **args)
  rows = [0, 1, 77, 127]
  check(eager[rows], *oracle(x[rows], **{k: v[rows] for k, v in c.items() if v is not None}))
  out = torch.zeros_like(X)
  torch.cuda.synchronize()
  g = torch.cuda.CUDAGraph()
  with torch.cuda.graph(g): ops().logit_rules(X, out=out, **args)
  for _ in range(2):
    out.zero_()
    g.replay()
    assert torch.equal(out, eager)
